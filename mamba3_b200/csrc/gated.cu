// Elementwise gated linear recurrence, forward and backward.
//
//   f_t = sigmoid(forget_t);  h_t = f_t h_{t-1} + (1 - f_t) value_t;  y_t = h_t silu(gate_t)
//
// per (batch, channel); without a gate y = h. Where reset_t is set, token t sees h_{t-1} = 0. The
// state and every product and sum are float32; y and the gradients are rounded once, to the
// activations' type. 1 - f is formed as sigmoid(-forget), not by subtraction: with f near 1 the
// subtraction would lose the time constant.
//
// Backward, with c_t = f_t (0 on a reset) and In_L = dstate, In_{t-1} = c_t G_t:
//   G_t = dy_t silu(gate_t) + In_t,            dvalue_t  = G_t (1 - f_t),
//   dforget_t = G_t (h_{t-1} - value_t) f_t (1 - f_t),   dgate_t = dy_t h_t silu'(gate_t),
//   dstate_0  = In_0.
#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "umma.cuh"

namespace m3 {

int report_error(int code, const char* msg);

// The error word of this unit's bounded waits, for m3_device_error(); the device is synchronised.
int read_gated_error(int clear) { return read_unit_error(clear); }

namespace {

using umma::mbar_expect_tx;
using umma::mbar_wait;
using umma::smem_u32;
using umma::tma_load3;

constexpr int kTile = 64;        // tokens a tile: the training forward keeps the state before each
constexpr int kChannels = 64;    // channels a CTA; a thread has two neighbouring ones
constexpr float kFloor = 1.4013e-45f;  // least product of decays without a reset, float32's least number: see fold()

template <typename T> constexpr bool kFine = std::is_same<T, float>::value;

// exp2 and reciprocal of the special-function unit, results below 2^-126 taken as 0. The compiler's __expf and
// __fdividef add the handling of such values, which no use here can tell apart.
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// With float32 inputs (kExact) a sigmoid is good to about one unit in the last place: the rounding of c log2(e), which
// for c = 8 is worth five units of its exponential, is recovered by fma, and the reciprocal gets a Newton step.
// Decays near 1 hold an error for as many tokens as they hold a value, so it shows in the state. 16-bit inputs, whose
// outputs are rounded to 8 or 11 bits, take the two instructions as they are.
template <bool kExact> __device__ __forceinline__ float exp_minus(float c) {
  const float t = c * -kLog2e, e = ex2_approx(t);
  if constexpr (!kExact) return e;
  constexpr float kLow = (float)(1.4426950408889634 - (double)kLog2e), kLn2 = 0.6931471805599453f;
  return fmaf(e, kLn2 * fmaf(c, -kLow, fmaf(c, -kLog2e, -t)), e);
}
template <bool kExact> __device__ __forceinline__ float reciprocal(float d) {
  const float r = rcp_approx(d);
  return kExact ? fmaf(r, fmaf(-d, r, 1.0f), r) : r;
}
__device__ __forceinline__ float at_least(float x, float least) {  // NaN stays NaN
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(least));
  return x;
}
__device__ __forceinline__ float at_most(float x, float most) {
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(most));
  return x;
}

// f = sigmoid(x) and 1 - f = sigmoid(-x). exp(-x) is kept at 2^125 or less, so that its reciprocal is no subnormal number
// (x at -125 ln 2 = -86.6 or more), and what f is there, 2^-125, is taken off every f: a masked logit (the type's lowest
// value, an infinity) drops a state of any size, and f is itself wherever it is not below 2^-100. NaN stays NaN.
// (kExact: past 100, where exp(-x) is 0, the differences of infinities are kept out.)
template <bool kExact> __device__ __forceinline__ void keep_lose(float x, float& keep, float& lose) {
  constexpr float kLeast = -86.643394f, kAtLeast = kExact ? 2.3509960e-38f /* exp(kLeast) */ : 2.3509887e-38f /* 2^-125 */;
  float e;
  if constexpr (kExact) e = exp_minus<true>(at_most(at_least(x, kLeast), 100.0f));
  else e = ex2_approx(at_most(x * -kLog2e, 125.0f));
  const float f = reciprocal<kExact>(1.0f + e);
  keep = f - kAtLeast;
  lose = e * f;
}

// sigmoid(x), 0 below -88.
template <bool kExact> __device__ __forceinline__ float sigmoid(float x) {
  if (kExact) x = at_most(at_least(x, -88.0f), 100.0f);
  return reciprocal<kExact>(1.0f + exp_minus<kExact>(x));
}

// A run of tokens as a map of the state before it: h -> a h + h0. a is exactly 0 where a reset lies in the run,
// and then nothing of h passes, not even an infinity or NaN; otherwise a product of decays is kept at kFloor or
// more, so that an infinity or NaN before the run does pass.
__device__ __forceinline__ float fold(float a, float h0, float h) { return a == 0.0f ? h0 : fmaf(a, h, h0); }
__device__ __forceinline__ float2 fold(float4 m, float2 h) { return make_float2(fold(m.x, m.z, h.x), fold(m.y, m.w, h.y)); }

// ---- two neighbouring values ---------------------------------------------------------------------

template <typename T> struct Two;
template <> struct Two<float> {
  using word = float2;
  static __device__ __forceinline__ float2 open(float2 w) { return w; }
  static __device__ __forceinline__ float2 close(float2 v) { return v; }
};
template <> struct Two<__half> {
  using word = __half2;
  static __device__ __forceinline__ float2 open(__half2 w) { return __half22float2(w); }
  static __device__ __forceinline__ __half2 close(float2 v) { return __float22half2_rn(v); }
};
template <> struct Two<__nv_bfloat16> {
  using word = __nv_bfloat162;
  static __device__ __forceinline__ float2 open(__nv_bfloat162 w) { return __bfloat1622float2(w); }
  static __device__ __forceinline__ __nv_bfloat162 close(float2 v) { return __float22bfloat162_rn(v); }
};

// A block's sequence: sequences lie along the grid's y, and its z where they are more than y may have.
__device__ __forceinline__ int sequence() { return blockIdx.z * gridDim.y + blockIdx.y; }

// ---- tiles ---------------------------------------------------------------------------------------

// Tokens t0 .. t0 + 63 of channels c0 .. c0 + 63 to a tile [64][64], for inputs that TMA cannot read: any
// strides; what is outside reads as 0.
template <typename T, int kThreads>
__device__ __forceinline__ void load_tile(T* tile, const m3_tensor& from, int b, int64_t t0, int c0, int64_t length, int channels) {
  const T* base = static_cast<const T*>(from.data) + b * from.stride[0];
#pragma unroll 16
  for (int i = threadIdx.x; i < kTile * kChannels; i += kThreads) {
    const int t = i / kChannels, c = i % kChannels;
    tile[i] = t0 + t < length && c0 + c < channels ? base[(t0 + t) * from.stride[1] + (c0 + c) * from.stride[2]]
                                                    : from_f<T>(0.0f);
  }
}

// The tiles of one tensor's channels: a tensor map [B][L][C] where TMA reads it.
struct Maps {
  CUtensorMap map[4];
};

template <typename T> __device__ __forceinline__ float2 read_two(const T* tile, int token, int lane) {
  return Two<T>::open(reinterpret_cast<const typename Two<T>::word*>(tile + token * kChannels)[lane]);
}

// Where a thread's two channels of its run's tokens go in an output: `at` is the CTA's tile, the same for all threads,
// and the rest an offset in 32 bits (kVec: 64 token strides fit them).
template <typename T, bool kVec> struct Rows {
  T* at;
  int64_t stride, channel_stride;
  uint32_t first;
  int c, channels;

  __device__ __forceinline__ void start(const m3_tensor& t, int b, int64_t token, int c0, int run0, int lane, int channels_) {
    at = static_cast<T*>(t.data) + b * t.stride[0] + token * t.stride[1] + c0 * t.stride[2];
    stride = t.stride[1];
    channel_stride = t.stride[2];
    c = c0 + 2 * lane;
    channels = channels_;
    first = kVec ? (uint32_t)run0 * (uint32_t)stride + 2 * lane : 0;
    if (!kVec) at += run0 * stride + 2 * lane * channel_stride;
  }
  __device__ __forceinline__ void go(int64_t tokens) { at += tokens * stride; }
  __device__ __forceinline__ void write(int j, float2 v) const {
    if constexpr (kVec) {  // both channels exist, or neither
      if (c < channels) *reinterpret_cast<typename Two<T>::word*>(at + (first + (uint32_t)j * (uint32_t)stride)) = Two<T>::close(v);
    } else {
      T* p = at + j * stride;
      if (c < channels) p[0] = from_f<T>(v.x);
      if (c + 1 < channels) p[channel_stride] = from_f<T>(v.y);
    }
  }
};

// Whether token t + lane of this warp's run of `run` tokens is a reset. Read a tile ahead.
__device__ __forceinline__ bool read_reset(const m3_tensor& reset, int b, int64_t t, int64_t length, int lane, int run) {
  return reset.data && lane < run && t + lane < length &&
         static_cast<const uint8_t*>(reset.data)[b * reset.stride[0] + (t + lane) * reset.stride[1]] != 0;
}

__device__ __forceinline__ float2 read_state(const m3_tensor& s, int b, int c, int channels) {
  const float* p = static_cast<const float*>(s.data);
  float2 v = make_float2(0.0f, 0.0f);
  if (p && c < channels) v.x = p[b * s.stride[0] + c * s.stride[1]];
  if (p && c + 1 < channels) v.y = p[b * s.stride[0] + (c + 1) * s.stride[1]];
  return v;
}
__device__ __forceinline__ void write_state(const m3_tensor& s, int b, int c, int channels, float2 v) {
  float* p = static_cast<float*>(s.data);
  if (c < channels) p[b * s.stride[0] + c * s.stride[1]] = v.x;
  if (c + 1 < channels) p[b * s.stride[0] + (c + 1) * s.stride[1]] = v.y;
}

// ---- clusters ------------------------------------------------------------------------------------
// The CTAs of a cluster take neighbouring tiles of the same channels, and go on together to the next ones.
// Each leaves its tile's map in every CTA's shared memory.

__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Send 16 bytes to the same place in the shared memory of CTA `rank`, counted there by the mbarrier at `bar`. No
// fence is involved: a cluster barrier's release would wait for every store to global memory before it.
__device__ __forceinline__ void send(int rank, uint32_t to, uint32_t bar, float4 v) {
  uint32_t there, counted;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(to), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(counted) : "r"(bar), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(there),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)), "r"(__float_as_uint(v.w)),
               "r"(counted)
               : "memory");
}

constexpr int kMaxCluster = 16;

// Shared memory of a CTA: kStages buffers of its tensors' tiles, the maps of its warps' runs (float4 = a, a', h0, h0'
// of a lane's two channels; the backward has a second set for In), in clusters the maps of the cluster's tiles for
// even and odd groups, the running state of 64 channels, an mbarrier for each stage and two for the exchange.
constexpr int kStages = 2;  // a power of two
template <typename T> __host__ __device__ constexpr int tile_bytes() { return kTile * kChannels * (int)sizeof(T); }
__host__ __device__ constexpr int smem_bytes(int tile_bytes, int tensors, int maps, int cluster) {
  return kStages * tensors * tile_bytes + (maps + (cluster > 1 ? 2 * cluster : 0)) * 32 * 16 + 32 * 8 + (kStages + 2) * 8;
}

// The exchange of a cluster: step i, every CTA leaves its tile's map in every CTA, maps[rank][lane], for even and odd
// steps apart. A CTA sends in step i + 2, over step i's maps, only when it has everyone's of step i + 1, and those
// were sent after their senders had read step i's.
struct Exchange {
  float4* maps;
  uint32_t bars;
  int rank, cluster;

  __device__ __forceinline__ void start() {
    if (threadIdx.x == 0) {
      for (int s = 0; s < 2; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * s));
      asm volatile("fence.mbarrier_init.release.cluster;");
    }
    __syncthreads();
    cluster_arrive();  // the others have started, and their barriers are there
    cluster_wait();
  }
  // `all`: warp 0's lanes have the tile's map. Returns the step's maps.
  __device__ __forceinline__ const float4* run(int64_t i, int warp, int lane, float4 all, bool& ok) {
    float4* at = maps + (i & 1) * cluster * 32;
    const uint32_t bar = bars + 8 * (uint32_t)(i & 1);
    if (threadIdx.x == 0) mbar_expect_tx(bar, (uint32_t)cluster * 32 * 16);
    if (warp == 0)
      for (int r = 0; r < cluster; ++r) send(r, smem_u32(at + rank * 32 + lane), bar, all);
    if (ok) ok = mbar_wait(bar, (uint32_t)(i >> 1) & 1u);
    __syncwarp();
    return at;
  }
  // No CTA leaves while another could still send to it (after a wait that gave up).
  __device__ __forceinline__ void finish() {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
};

// The map of one run after another.
__device__ __forceinline__ void join(float4& m, float4 next) {
  m.z = fold(next.x, next.z, m.z);
  m.w = fold(next.y, next.w, m.w);
  m.x = m.x == 0.0f || next.x == 0.0f ? 0.0f : fmaxf(m.x * next.x, kFloor);
  m.y = m.y == 0.0f || next.y == 0.0f ? 0.0f : fmaxf(m.y * next.y, kFloor);
}

// What both kernels are made of: a CTA's channels and tiles, and the copies of the tiles into shared memory, kStages
// deep. The tiles come in groups of `cluster`; step i is the i-th group that the kernel takes.
template <typename T, int kTensors, int kThreads, bool kVec> struct Pipeline {
  T* tiles;
  uint32_t bars;  // shared-memory address of the stages' mbarriers
  int64_t ntiles, groups;
  int64_t newest = -1;  // the last step loaded
  bool ok = true;

  __device__ __forceinline__ void start(T* at, uint32_t bar) {
    tiles = at;
    bars = bar;
    if constexpr (kVec) {
      if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + 8 * s));
        asm volatile("fence.mbarrier_init.release.cluster;");
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ T* stage(int64_t i) { return tiles + (i & (kStages - 1)) * kTensors * kTile * kChannels; }
  // Start on step i's tile t; everyone is done with the stage.
  __device__ __forceinline__ void load(const Maps& maps, const m3_tensor* const* from, int64_t i, int64_t t, int b, int c0,
                                       const m3_gated_args& a) {
    if (t < 0 || t >= ntiles || !ok) return;
    newest = i;
    T* to = stage(i);
    if constexpr (kVec) {
      if (threadIdx.x == 0) {
        const uint32_t bar = bars + 8 * (uint32_t)(i & (kStages - 1));
        mbar_expect_tx(bar, kTensors * tile_bytes<T>());
#pragma unroll
        for (int k = 0; k < kTensors; ++k)
          tma_load3(smem_u32(to + k * kTile * kChannels), &maps.map[k], c0, (int)(t * kTile), b, bar);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kTensors; ++k)
        load_tile<T, kThreads>(to + k * kTile * kChannels, *from[k], b, t * kTile, c0, a.length, a.channels);
    }
  }
  // Step i's tile is there; everyone is done with the step before. A wait that gave up (the error word says so) is not
  // repeated: what is left runs through without it.
  __device__ __forceinline__ const T* ready(int64_t i, int64_t t) {
    if constexpr (kVec) {
      if (threadIdx.x < 32 && ok && t < ntiles)  // the barrier after it passes it on to the other warps
        ok = mbar_wait(bars + 8 * (uint32_t)(i & (kStages - 1)), (uint32_t)(i / kStages) & 1u);
    }
    __syncthreads();
    return stage(i);
  }
  // After a wait that gave up: the copies still under way land before the block's shared memory goes.
  __device__ __forceinline__ void finish() {
    if constexpr (kVec) {
      if (threadIdx.x == 0 && !ok)
        for (int64_t i = newest - kStages + 1; i <= newest; ++i)
          if (i >= 0) mbar_wait(bars + 8 * (uint32_t)(i & (kStages - 1)), (uint32_t)(i / kStages) & 1u);
    }
  }
};

// The first pass over a run: decays f, inputs (1 - f) value (kLose: 1 - f alone) and the run's map. kWhole: every
// token is there and none is a reset.
template <typename T, bool kWhole, bool kLose, int kRun>
__device__ __forceinline__ float4 open_run(const T* forget, const T* value, int token, int lane, int n, uint32_t resets,
                                           float2 (&keep)[kRun], float2 (&other)[kRun]) {
  float4 m = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
  bool reset = false;
#pragma unroll
  for (int j = 0; j < kRun; ++j) {
    if (!kWhole && j >= n) {
      keep[j] = make_float2(1.0f, 1.0f);
      other[j] = make_float2(0.0f, 0.0f);
      continue;
    }
    const float2 f = read_two(forget, token + j, lane), v = read_two(value, token + j, lane);
    float2 lose;
    keep_lose<kFine<T>>(f.x, keep[j].x, lose.x);
    keep_lose<kFine<T>>(f.y, keep[j].y, lose.y);
    const float2 in = make_float2(lose.x * v.x, lose.y * v.y);
    other[j] = kLose ? lose : in;
    if (!kWhole && (resets >> j & 1u)) {
      m.z = m.w = 0.0f;
      reset = true;
    }
    m.z = fmaf(keep[j].x, m.z, in.x);
    m.w = fmaf(keep[j].y, m.w, in.y);
    m.x *= keep[j].x;
    m.y *= keep[j].y;
  }
  m.x = reset ? 0.0f : fmaxf(m.x, kFloor);
  m.y = reset ? 0.0f : fmaxf(m.y, kFloor);
  return m;
}

// Forward. One pass over the inputs: a thread folds its run of 16 tokens into a map (a, h0), the maps of the 4 runs
// of a tile (and of a cluster's tiles) give every run the state before it, and the run is repeated from there
// out of registers. CTAs walk a sequence's tiles one after another; where sequences and channels are too few to
// fill the GPU, a cluster walks them together. Every input is read once and nothing but y, the last state and, for a
// backward pass, a state a tile is written.
// bf16 with a gate: 8 x 8192 x 2048 in 227 us (4.7 TB/s, 73 % of a copy), 4 x 2048 x 2048 in 39, 1 x 65536 x 1536 in 264.
// On full grids nothing is at its limit: 128 registers a thread leave sixteen warps an SM, whose chains of dependent
// instructions fill 56 % of the issue slots, the special-function unit (two exp2 and two reciprocals a value) half and
// DRAM's rate to 36 % (4 x 2048 x 2048). Few channels wait for the exchange of a cluster's maps, step after step. Runs of
// 16 tokens halve the folding that runs of 8 need.
constexpr int kFwdWarps = 4, kFwdThreads = 32 * kFwdWarps, kFwdRun = kTile / kFwdWarps;

template <typename T, bool kGate, bool kVec>
__global__ void __launch_bounds__(kFwdThreads, 4)
    gated_fwd_kernel(const __grid_constant__ Maps maps, const m3_gated_args a, const int cluster) {
  constexpr int kTensors = kGate ? 3 : 2, kElems = kTile * kChannels, kRun = kFwdRun, kWarps = kFwdWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  float4* runs = reinterpret_cast<float4*>(smem + kStages * kTensors * tile_bytes<T>());
  float4* peers = runs + kWarps * 32;
  float2* next = reinterpret_cast<float2*>(peers + (cluster > 1 ? 2 * cluster * 32 : 0));  // the state after the tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? cluster_rank() : 0;
  const int b = sequence(), c0 = blockIdx.x / cluster * kChannels, c = c0 + 2 * lane;
  if (b >= a.batch) return;  // as the whole cluster does
  Pipeline<T, kTensors, kFwdThreads, kVec> pipe;
  pipe.ntiles = (a.length + kTile - 1) / kTile;
  pipe.groups = (pipe.ntiles + cluster - 1) / cluster;
  pipe.start(reinterpret_cast<T*>(smem), smem_u32(next + 32));
  const m3_tensor* from[3] = {&a.forget, &a.value, &a.gate};
  for (int i = 0; i < kStages - 1; ++i) pipe.load(maps, from, i, i * cluster + rank, b, c0, a);
  float2 carry = read_state(a.state, b, c, a.channels);  // the state before the group of tiles
  bool flag = read_reset(a.reset, b, (int64_t)rank * kTile + warp * kRun, a.length, lane, kRun);
  Rows<T, kVec> y;
  y.start(a.y, b, (int64_t)rank * kTile, c0, warp * kRun, lane, a.channels);
  Exchange exchange{peers, smem_u32(next + 32) + 8 * kStages, rank, cluster};
  if (cluster > 1) exchange.start();
  for (int64_t g = 0; g < pipe.groups; ++g, y.go(cluster * kTile)) {
    const int64_t t = g * cluster + rank, t0 = t * kTile + warp * kRun;
    const uint32_t resets = __ballot_sync(0xffffffffu, flag);
    flag = read_reset(a.reset, b, t0 + (int64_t)cluster * kTile, a.length, lane, kRun);
    const T* tile = pipe.ready(g, t);
    if (cluster == 1 && g > 0) carry = next[lane];
    pipe.load(maps, from, g + kStages - 1, t + (kStages - 1) * cluster, b, c0, a);
    const int n = t0 >= a.length ? 0 : a.length - t0 < kRun ? (int)(a.length - t0) : kRun;  // tokens of this run
    const bool whole = n == kRun && resets == 0;
    float2 keep[kRun], in[kRun];
    const float4 map = whole ? open_run<T, true, false>(tile, tile + kElems, warp * kRun, lane, n, resets, keep, in)
                             : open_run<T, false, false>(tile, tile + kElems, warp * kRun, lane, n, resets, keep, in);
    runs[warp * 32 + lane] = map;
    __syncthreads();
    float2 h = carry;  // the state before this CTA's tile
    if (cluster > 1) {
      float4 all = runs[lane];
      if (warp == 0)
        for (int w = 1; w < kWarps; ++w) join(all, runs[w * 32 + lane]);
      const float4* of = exchange.run(g, warp, lane, all, pipe.ok);
      for (int r = 0; r < cluster; ++r) {
        if (r == rank) h = carry;
        carry = fold(of[r * 32 + lane], carry);
      }
    }
    if (a.carry.data && warp == 0 && t < pipe.ntiles) {
      float* kept = static_cast<float*>(a.carry.data) + b * a.carry.stride[0] + t * a.carry.stride[1];
      if (c < a.channels) kept[c] = h.x;
      if (c + 1 < a.channels) kept[c + 1] = h.y;
    }
    for (int w = 0; w < warp; ++w) h = fold(runs[w * 32 + lane], h);
    if (cluster == 1 && warp == kWarps - 1) next[lane] = fold(map, h);
    auto finish = [&](int j) {
      h.x = fmaf(keep[j].x, h.x, in[j].x);
      h.y = fmaf(keep[j].y, h.y, in[j].y);
      float2 out = h;
      if constexpr (kGate) {
        const float2 q = read_two(tile + 2 * kElems, warp * kRun + j, lane);
        out.x *= q.x * sigmoid<kFine<T>>(q.x);
        out.y *= q.y * sigmoid<kFine<T>>(q.y);
      }
      y.write(j, out);
    };
    if (whole) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) finish(j);
    } else {
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (j >= n) break;
        if (resets >> j & 1u) h = make_float2(0.0f, 0.0f);
        finish(j);
      }
    }
  }
  pipe.finish();
  if (cluster > 1) exchange.finish();
  else {
    __syncthreads();
    carry = next[lane];
  }
  if (rank == 0 && warp == 0) write_state(a.out_state, b, c, a.channels, carry);
}

// Backward, the tiles from the last to the first: the states of a tile come from the state kept before it, as in
// the forward, and the gradients In run back through maps of the same a with h0 of their own.
// bf16 with a gate: 8 x 8192 x 2048 in 577 us (3.3 TB/s, 50 % of a copy), 4 x 2048 x 2048 in 92, 1 x 65536 x 1536 in
// 590. Five pairs of values a token are held over the tile's barrier, 128 registers a thread for runs of 8, so four warps
// a scheduler: 57 % of the issue slots, DRAM's rate to 27 %, no pipe above 36 % (4 x 2048 x 2048); a warp waits most for
// the instruction before. Runs of 4 in 16 warps of 64 registers: 1002 us against 650 then; of 16 in four warps, slower too.
constexpr int kBwdWarps = 8, kBwdThreads = 32 * kBwdWarps, kBwdRun = kTile / kBwdWarps;

template <typename T, bool kGate, bool kVec>
__global__ void __launch_bounds__(kBwdThreads, 2)
    gated_bwd_kernel(const __grid_constant__ Maps maps, const m3_gated_args a, const int cluster) {
  constexpr int kTensors = kGate ? 4 : 3, kElems = kTile * kChannels, kRun = kBwdRun, kWarps = kBwdWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  float4* runs = reinterpret_cast<float4*>(smem + kStages * kTensors * tile_bytes<T>());
  float4* back = runs + kWarps * 32;  // (a, a', In0, In0') of the runs from the back
  float4* peers = back + kWarps * 32;
  float2* next = reinterpret_cast<float2*>(peers + (cluster > 1 ? 2 * cluster * 32 : 0));  // In before the tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? cluster_rank() : 0;
  const int b = sequence(), c0 = blockIdx.x / cluster * kChannels, c = c0 + 2 * lane;
  if (b >= a.batch) return;  // as the whole cluster does
  Pipeline<T, kTensors, kBwdThreads, kVec> pipe;
  pipe.ntiles = (a.length + kTile - 1) / kTile;
  pipe.groups = (pipe.ntiles + cluster - 1) / cluster;
  pipe.start(reinterpret_cast<T*>(smem), smem_u32(next + 32));
  const m3_tensor* from[4] = {&a.forget, &a.value, &a.dy, &a.gate};
  const int64_t last = (pipe.groups - 1) * cluster + rank;  // this CTA's tile of step 0; step i has last - i * cluster
  // Only the first step's tile can be past the end. It is not loaded, so the stages' mbarriers do not count it: the
  // pipeline's steps start at `skipped`.
  const int skipped = last >= pipe.ntiles ? 1 : 0;
  for (int i = 0; i < kStages - 1; ++i) pipe.load(maps, from, i - skipped, last - i * cluster, b, c0, a);
  auto before = [&](int64_t t) {  // the state kept before tile t
    float2 h = make_float2(0.0f, 0.0f);
    if (t >= 0 && t < pipe.ntiles) {
      const float* kept = static_cast<const float*>(a.carry.data) + b * a.carry.stride[0] + t * a.carry.stride[1];
      if (c < a.channels) h.x = kept[c];
      if (c + 1 < a.channels) h.y = kept[c + 1];
    }
    return h;
  };
  float2 carry = read_state(a.dstate, b, c, a.channels);  // In after the group of tiles
  bool flag = read_reset(a.reset, b, last * kTile + warp * kRun, a.length, lane, kRun);
  float2 kept = before(last);
  Rows<T, kVec> dvalue, dforget, dgate;
  dvalue.start(a.dvalue, b, last * kTile, c0, warp * kRun, lane, a.channels);
  dforget.start(a.dforget, b, last * kTile, c0, warp * kRun, lane, a.channels);
  if constexpr (kGate) dgate.start(a.dgate, b, last * kTile, c0, warp * kRun, lane, a.channels);
  Exchange exchange{peers, smem_u32(next + 32) + 8 * kStages, rank, cluster};
  if (cluster > 1) exchange.start();
  for (int64_t i = 0; i < pipe.groups; ++i) {
    const int64_t t = last - i * cluster, t0 = t * kTile + warp * kRun;
    const uint32_t resets = __ballot_sync(0xffffffffu, flag);
    float2 h = kept;
    if (i + 1 < pipe.groups) {
      flag = read_reset(a.reset, b, t0 - (int64_t)cluster * kTile, a.length, lane, kRun);
      kept = before(t - cluster);
    }
    const T* tile = pipe.ready(i - skipped, t);
    if (cluster == 1 && i > 0) carry = next[lane];
    pipe.load(maps, from, i - skipped + kStages - 1, t - (kStages - 1) * cluster, b, c0, a);
    const int n = t0 >= a.length ? 0 : a.length - t0 < kRun ? (int)(a.length - t0) : kRun;
    const bool whole = n == kRun && resets == 0;
    float2 keep[kRun], lose[kRun], dh[kRun], slope[kRun];  // dy silu(gate), dy silu'(gate)
    const float4 map = whole ? open_run<T, true, true>(tile, tile + kElems, warp * kRun, lane, n, resets, keep, lose)
                             : open_run<T, false, true>(tile, tile + kElems, warp * kRun, lane, n, resets, keep, lose);
    float4 rmap = make_float4(map.x, map.y, 0.0f, 0.0f);
#pragma unroll
    for (int j = kRun - 1; j >= 0; --j) {
      dh[j] = slope[j] = make_float2(0.0f, 0.0f);
      if (!whole && j >= n) continue;
      dh[j] = read_two(tile + 2 * kElems, warp * kRun + j, lane);
      if constexpr (kGate) {
        const float2 q = read_two(tile + 3 * kElems, warp * kRun + j, lane);
        const float2 sig = make_float2(sigmoid<kFine<T>>(q.x), sigmoid<kFine<T>>(q.y));
        const float2 qs = make_float2(q.x * sig.x, q.y * sig.y);  // silu' = s + gate s (1 - s)
        slope[j] = make_float2(dh[j].x * fmaf(qs.x, 1.0f - sig.x, sig.x), dh[j].y * fmaf(qs.y, 1.0f - sig.y, sig.y));
        dh[j].x *= qs.x;
        dh[j].y *= qs.y;
      }
      rmap.z = keep[j].x * (dh[j].x + rmap.z);
      rmap.w = keep[j].y * (dh[j].y + rmap.w);
      if (!whole && (resets >> j & 1u)) rmap.z = rmap.w = 0.0f;
    }
    runs[warp * 32 + lane] = map;
    back[warp * 32 + lane] = rmap;
    __syncthreads();
    float2 mine = carry;  // In after this CTA's tile, then after this run
    if (cluster > 1) {
      float4 all = back[(kWarps - 1) * 32 + lane];
      if (warp == 0)
        for (int w = kWarps - 2; w >= 0; --w) join(all, back[w * 32 + lane]);
      const float4* of = exchange.run(i, warp, lane, all, pipe.ok);
      for (int r = cluster - 1; r >= 0; --r) {
        if (r == rank) mine = carry;
        carry = fold(of[r * 32 + lane], carry);
      }
    }
    for (int w = 0; w < warp; ++w) h = fold(runs[w * 32 + lane], h);
    for (int w = kWarps - 1; w > warp; --w) mine = fold(back[w * 32 + lane], mine);
    if (cluster == 1 && warp == 0) next[lane] = fold(rmap, mine);
    const float2 h_in = h;
    float2 after[kRun];  // h_t
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (!whole && j >= n) break;
      if (!whole && (resets >> j & 1u)) h = make_float2(0.0f, 0.0f);
      const float2 v = read_two(tile + kElems, warp * kRun + j, lane);
      h.x = fmaf(keep[j].x, h.x, lose[j].x * v.x);
      h.y = fmaf(keep[j].y, h.y, lose[j].y * v.y);
      after[j] = h;
    }
    auto finish = [&](int j, float2 prev) {  // prev: h_{t-1} as token t sees it
      const float2 v = read_two(tile + kElems, warp * kRun + j, lane);
      if constexpr (kGate) dgate.write(j, make_float2(slope[j].x * after[j].x, slope[j].y * after[j].y));
      const float2 G = make_float2(dh[j].x + mine.x, dh[j].y + mine.y);
      const float2 dv = make_float2(G.x * lose[j].x, G.y * lose[j].y);
      mine.x = keep[j].x * G.x;
      mine.y = keep[j].y * G.y;
      dvalue.write(j, dv);
      dforget.write(j, make_float2(mine.x * lose[j].x * (prev.x - v.x), mine.y * lose[j].y * (prev.y - v.y)));
    };
    if (whole) {
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) finish(j, j ? after[j - 1] : h_in);
    } else {
#pragma unroll
      for (int j = kRun - 1; j >= 0; --j) {
        if (j >= n) continue;
        const bool fresh = resets >> j & 1u;
        finish(j, fresh ? make_float2(0.0f, 0.0f) : j ? after[j - 1] : h_in);
        if (fresh) mine = make_float2(0.0f, 0.0f);
      }
    }
    dvalue.go(-cluster * kTile);
    dforget.go(-cluster * kTile);
    if constexpr (kGate) dgate.go(-cluster * kTile);
  }
  pipe.finish();
  if (cluster > 1) exchange.finish();
  else {
    __syncthreads();
    carry = next[lane];
  }
  if (a.dinitial.data && rank == 0 && warp == 0) write_state(a.dinitial, b, c, a.channels, carry);
}

// One token: nothing but elementwise work, one thread for kWide neighbouring channels. 256 x 5120 in bf16 takes 4.2 us
// (76 % of a copy), 1 x 5120 1.4 in a graph: a launch, and the latency of one load.
template <typename T, int kWide>
__global__ void __launch_bounds__(128) gated_step_kernel(const m3_gated_args a) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * kWide, b = sequence();
  if (c >= a.channels || b >= a.batch) return;
  auto at = [&](const m3_tensor& t) { return static_cast<T*>(t.data) + b * t.stride[0] + c * t.stride[2]; };
  float h[kWide], f[kWide], v[kWide], q[kWide], y[kWide];
  auto get = [&](const T* p, float* to) {
    alignas(16) T w[kWide];
    if constexpr (kWide == 4 && sizeof(T) == 4) *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(p);
    else if constexpr (kWide == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else w[0] = *p;
#pragma unroll
    for (int e = 0; e < kWide; ++e) to[e] = to_f(w[e]);
  };
  const float* sp = static_cast<const float*>(a.state.data) + b * a.state.stride[0] + c * a.state.stride[1];
#pragma unroll
  for (int e = 0; e < kWide; ++e) h[e] = q[e] = 0.0f;
  if (a.state.data) {
    if constexpr (kWide == 4) *reinterpret_cast<float4*>(h) = *reinterpret_cast<const float4*>(sp);
    else h[0] = *sp;
  }
  get(at(a.forget), f);
  get(at(a.value), v);
  if (a.gate.data) get(at(a.gate), q);
  if (a.carry.data) {
#pragma unroll
    for (int e = 0; e < kWide; ++e) static_cast<float*>(a.carry.data)[b * a.carry.stride[0] + c + e] = h[e];
  }
  const bool reset = a.reset.data && static_cast<const uint8_t*>(a.reset.data)[b * a.reset.stride[0]] != 0;
#pragma unroll
  for (int e = 0; e < kWide; ++e) {
    float keep, lose;
    keep_lose<kFine<T>>(f[e], keep, lose);
    h[e] = fmaf(keep, reset ? 0.0f : h[e], lose * v[e]);
    y[e] = a.gate.data ? h[e] * (q[e] * sigmoid<kFine<T>>(q[e])) : h[e];
  }
  float* op = static_cast<float*>(a.out_state.data) + b * a.out_state.stride[0] + c * a.out_state.stride[1];
  T* yp = at(a.y);
  if constexpr (kWide == 4) {
    *reinterpret_cast<float4*>(op) = *reinterpret_cast<const float4*>(h);
    alignas(16) T w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = from_f<T>(y[e]);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(yp) = *reinterpret_cast<const float4*>(w);
    else *reinterpret_cast<uint2*>(yp) = *reinterpret_cast<const uint2*>(w);
  } else {
    *op = h[0];
    *yp = from_f<T>(y[0]);
  }
}

// ---- host ----------------------------------------------------------------------------------------

// A grid of `blocks` for each sequence; see sequence().
dim3 sequences_grid(int64_t blocks, int batch) {
  const int z = (batch + 65534) / 65535;
  return dim3((unsigned)blocks, (unsigned)((batch + z - 1) / z), (unsigned)z);
}

// Rows of `bytes`-aligned runs of channels: unit stride, aligned start and aligned batch and token strides.
bool rows_aligned(const m3_tensor& t, int elem, int bytes) {
  return t.data == nullptr || (t.stride[2] == 1 && reinterpret_cast<uintptr_t>(t.data) % bytes == 0 &&
                               t.stride[0] * elem % bytes == 0 && t.stride[1] * elem % bytes == 0);
}

template <typename T> cudaError_t launch_step_token(const m3_gated_args& a, cudaStream_t stream) {
  constexpr int kElem = sizeof(T);
  auto state_aligned = [](const m3_tensor& t) {
    return t.data == nullptr || (t.stride[1] == 1 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && t.stride[0] % 4 == 0);
  };
  const bool wide = a.channels % 4 == 0 && rows_aligned(a.value, kElem, 4 * kElem) && rows_aligned(a.forget, kElem, 4 * kElem) &&
                    rows_aligned(a.gate, kElem, 4 * kElem) && rows_aligned(a.y, kElem, 4 * kElem) && state_aligned(a.state) &&
                    state_aligned(a.out_state);
  const int per_block = 128 * (wide ? 4 : 1);
  const dim3 grid = sequences_grid((a.channels + per_block - 1) / per_block, a.batch);
  if (wide) gated_step_kernel<T, 4><<<grid, 128, 0, stream>>>(a);
  else gated_step_kernel<T, 1><<<grid, 128, 0, stream>>>(a);
  return cudaGetLastError();
}

// Whether TMA can read a tensor's tiles: unit stride along the channels, rows and start on 16 bytes.
bool tma_reads(const m3_tensor& t, const m3_gated_args& a, int elem) {
  auto whole = [&](int64_t stride, int64_t extent) { return extent == 1 || (stride > 0 && stride * elem % 16 == 0); };
  return t.data == nullptr || (t.stride[2] == 1 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && whole(t.stride[0], a.batch) &&
                               whole(t.stride[1], a.length) && a.length < INT32_MAX - kTile);
}

// Whether two neighbouring channels can be written as one word, a tile of 64 tokens within offsets of 32 bits.
bool pairs_written(const m3_tensor& t, const m3_gated_args& a, int elem) {
  return t.data == nullptr || (a.channels % 2 == 0 && rows_aligned(t, elem, 2 * elem) && t.stride[1] >= 0 && t.stride[1] < (1 << 23));
}

bool encode(CUtensorMap* map, const m3_tensor& t, const m3_gated_args& a, int elem) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const int64_t row = ((int64_t)a.channels * elem + 15) / 16 * 16;  // a stride that is never used
  const int64_t token = a.length == 1 ? row : t.stride[1] * elem;
  const cuuint64_t dims[3] = {(cuuint64_t)a.channels, (cuuint64_t)a.length, (cuuint64_t)a.batch};
  const cuuint64_t strides[2] = {(cuuint64_t)token, (cuuint64_t)(a.batch == 1 ? row : t.stride[0] * elem)};
  const cuuint32_t box[3] = {kChannels, kTile, 1}, step[3] = {1, 1, 1};
  const CUtensorMapDataType type = t.dtype == M3_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : t.dtype == M3_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(map, type, 3, t.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool kGate, bool kVec, bool kBackward> auto pass_kernel() {
  if constexpr (kBackward) return gated_bwd_kernel<T, kGate, kVec>;
  else return gated_fwd_kernel<T, kGate, kVec>;
}

// How a pass lies in a CTA.
template <typename T, bool kGate, bool kBackward> struct Pass {
  static constexpr int kThreads = kBackward ? kBwdThreads : kFwdThreads;
  static constexpr int smem(int cluster) {
    return smem_bytes(tile_bytes<T>(), (kBackward ? 3 : 2) + (kGate ? 1 : 0), kBackward ? 2 * kBwdWarps : kFwdWarps, cluster);
  }
  // CTAs of a cluster of `size` that an SM has room for: by shared memory, which grows with the cluster, and by registers
  // at the 128 that both kernels take.
  static constexpr int room(int size) { return std::min(227 * 1024 / (smem(size) + 1024), 65536 / (128 * kThreads)); }

  static cudaLaunchConfig_t config(dim3 grid, int cluster, cudaLaunchAttribute* attr, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem(cluster);
    cfg.stream = stream;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = cluster;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cfg;
  }
  // The limits are the kernel's, not the launch's: the largest cluster's always, or another thread with a shorter sequence
  // could lower them between this call and a launch.
  template <typename K> static cudaError_t raise_limits(K kernel) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem(kMaxCluster));
    return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }
  // Clusters of `size` that the device hosts at once, as it says itself: a cluster lies within a group of 16 to 20 SMs,
  // and what is left of a group holds none. Without a device, 148 SMs without groups.
  static int64_t hosted(int size) {
    static std::atomic<int> cached[64][kMaxCluster + 1];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) {
      std::atomic<int>& held = cached[dev][size];
      if (const int known = held.load(std::memory_order_relaxed)) return known - 1;
      const auto kernel = pass_kernel<T, kGate, true, kBackward>();
      cudaLaunchAttribute attr[1];
      const cudaLaunchConfig_t cfg = config(dim3(size), size, attr, nullptr);
      if (raise_limits(kernel) == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess) {
        held.store(n + 1, std::memory_order_relaxed);
        return n;
      }
    }
    cudaGetLastError();
    return size > 8 && room(size) < 2 ? 0 : (int64_t)sm_count() * room(size) / size;
  }
};

template <typename P> int cluster_size(const m3_gated_args& a) {
  const int64_t ntiles = (a.length + kTile - 1) / kTile;
  const int64_t blocks = (int64_t)a.batch * ((a.channels + kChannels - 1) / kChannels);
  // A cluster takes a sequence's tiles together while the device hosts all clusters at once: clusters of up to 4 in all the
  // room there is, larger ones, whose exchange takes as long as a tile, up to two CTAs an SM, and eights, where all their
  // tiles are under way from the start, in all the room too. Sixteens are the last power; tens stand where sixteens have no
  // such room. Measured in bf16 with a gate, forward and backward, us:
  //                                          2           4           8          10          16
  //   1 x 65536 x 1216   (19 x 64 channels)  932, 2060   472, 1060   294, 686   255, 578    203, 650
  //   1 x 65536 x 1536   (24)                933, 2072   473, 1064   298, 691   256, 583    318, 736
  //   1 x 65536 x 1856   (29)                933, 2076   473, 1071   303, 699   310, 1006   351, 995
  //   2 x 4096 x 1024    (32)                61.7, 133   32.8, 72.9  23.2, 48.9 24.7, 74.2  28.1, 71.4
  //   4 x 2048 x 1024    (64)                32.5, 69.0  22.0, 47.4  27.6, 51.7 27.6, 70.3  30.9, 71.4
  //   1 x 640 x 4736     (74)                12.5, 23.3  12.2, 31.0  16.4, 35.3 12.4, 25.1
  //   3 x 777 x 1001, float32, no gate (48)  34.1, 39.6  23.7, 32.1  16.7, 32.6 27.9, 66.8
  // What is not hosted at once runs in waves: tens of 29 (backward), fours of 74 (backward, 296 CTAs for 296 places).
  int cluster = 1;
  for (int size = 2; size <= kMaxCluster && size <= ntiles; size *= 2) {
    const bool all_room = size < 8 || (size == 8 && 8 * kStages >= ntiles);
    if (blocks > P::hosted(size) || (!all_room && size * blocks > 2 * (int64_t)sm_count())) break;
    cluster = size;
  }
  if (cluster == 8 && P::room(10) >= 2 && 10 <= ntiles && 10 * blocks <= 2 * (int64_t)sm_count() && blocks <= P::hosted(10)) cluster = 10;
  return cluster;
}

template <typename T, bool kGate, bool kBackward> cudaError_t launch_tiles(const m3_gated_args& a, const Maps& maps, bool vec, cudaStream_t stream) {
  using P = Pass<T, kGate, kBackward>;
  const int cluster = cluster_size<P>(a);
  const auto kernel = vec ? pass_kernel<T, kGate, true, kBackward>() : pass_kernel<T, kGate, false, kBackward>();
  const cudaError_t e = P::raise_limits(kernel);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  const dim3 grid = sequences_grid((int64_t)(a.channels + kChannels - 1) / kChannels * cluster, a.batch);
  const cudaLaunchConfig_t cfg = P::config(grid, cluster, attr, stream);
  return cudaLaunchKernelEx(&cfg, kernel, maps, a, cluster);
}

template <typename T> cudaError_t launch_fwd(const m3_gated_args& a, cudaStream_t stream) {
  if (a.length == 1) return launch_step_token<T>(a, stream);
  constexpr int kElem = sizeof(T);
  Maps maps = {};
  const bool vec = tma_reads(a.forget, a, kElem) && tma_reads(a.value, a, kElem) && tma_reads(a.gate, a, kElem) &&
                   pairs_written(a.y, a, kElem);
  if (vec && !(encode(&maps.map[0], a.forget, a, kElem) && encode(&maps.map[1], a.value, a, kElem) &&
               (a.gate.data == nullptr || encode(&maps.map[2], a.gate, a, kElem))))
    return cudaErrorInvalidValue;
  return a.gate.data ? launch_tiles<T, true, false>(a, maps, vec, stream) : launch_tiles<T, false, false>(a, maps, vec, stream);
}

template <typename T> cudaError_t launch_bwd(const m3_gated_args& a, cudaStream_t stream) {
  constexpr int kElem = sizeof(T);
  Maps maps = {};
  const bool vec = tma_reads(a.forget, a, kElem) && tma_reads(a.value, a, kElem) && tma_reads(a.dy, a, kElem) &&
                   tma_reads(a.gate, a, kElem) && pairs_written(a.dvalue, a, kElem) && pairs_written(a.dforget, a, kElem) &&
                   pairs_written(a.dgate, a, kElem);
  if (vec && !(encode(&maps.map[0], a.forget, a, kElem) && encode(&maps.map[1], a.value, a, kElem) &&
               encode(&maps.map[2], a.dy, a, kElem) && (a.gate.data == nullptr || encode(&maps.map[3], a.gate, a, kElem))))
    return cudaErrorInvalidValue;
  return a.gate.data ? launch_tiles<T, true, true>(a, maps, vec, stream) : launch_tiles<T, false, true>(a, maps, vec, stream);
}

bool shaped(const m3_tensor& t, int ndim, int dtype) { return t.data == nullptr || (t.ndim == ndim && t.dtype == dtype); }

int check(const m3_gated_args& a, bool backward) {
  if (a.batch <= 0 || a.length <= 0 || a.channels <= 0)
    return report_error(M3_ERR_SHAPE, "gated scan: batch, length and channels must be positive");
  constexpr int32_t kMost = INT32_MAX - 4096;  // channels past the last block's still count in 32 bits
  if (a.channels > kMost) return report_error(M3_ERR_SHAPE, "gated scan: channels above 2^31 - 4097");
  if (a.batch > INT32_MAX - 65536) return report_error(M3_ERR_SHAPE, "gated scan: batch above 2^31 - 65537");
  if (!a.value.data || !a.forget.data) return report_error(M3_ERR_ARGUMENT, "gated scan: value and forget are required");
  const int act = a.value.dtype;
  if (act != M3_F32 && act != M3_F16 && act != M3_BF16)
    return report_error(M3_ERR_DTYPE, "gated scan: activations must be float32, float16 or bfloat16");
  bool ok = shaped(a.value, 3, act) && shaped(a.forget, 3, act) && shaped(a.gate, 3, act) && shaped(a.reset, 2, M3_U8) &&
            shaped(a.state, 2, M3_F32) && shaped(a.carry, 3, M3_F32);
  if (!backward) {
    if (!a.y.data || !a.out_state.data) return report_error(M3_ERR_ARGUMENT, "gated scan: y and out_state are required");
    ok = ok && shaped(a.y, 3, act) && shaped(a.out_state, 2, M3_F32);
  } else {
    if (!a.dy.data || !a.carry.data || !a.dvalue.data || !a.dforget.data || (a.gate.data && !a.dgate.data))
      return report_error(M3_ERR_ARGUMENT, "gated scan backward: dy, carry and a gradient for each input are required");
    ok = ok && shaped(a.dy, 3, act) && shaped(a.dvalue, 3, act) && shaped(a.dforget, 3, act) && shaped(a.dgate, 3, act) &&
         shaped(a.dstate, 2, M3_F32) && shaped(a.dinitial, 2, M3_F32);
  }
  if (!ok) return report_error(M3_ERR_DTYPE, "gated scan: activations share one dtype, states are float32, reset is bytes");
  if (a.carry.data && a.carry.stride[2] != 1) return report_error(M3_ERR_LAYOUT, "gated scan: carry channels must be contiguous");
  if (a.device >= 0 && cudaSetDevice(a.device) != cudaSuccess)
    return report_error(M3_ERR_CUDA, "gated scan: cannot select the device");
  return M3_OK;
}

int launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return M3_OK;
  return report_error(M3_ERR_CUDA, (std::string(what) + " launch failed: " + cudaGetErrorString(e)).c_str());
}

}  // namespace
}  // namespace m3

extern "C" int m3_gated_tile(void) { return m3::kTile; }

extern "C" int m3_gated_cluster(const m3_gated_args* args, int backward) {
  using namespace m3;
  if (args == nullptr || args->batch <= 0 || args->length <= 0 || args->channels <= 0) return 0;
  if (args->length == 1 && !backward) return 1;
  auto of = [&](auto type) {  // 16-bit types lie alike
    using T = decltype(type);
    if (args->gate.data) return backward ? cluster_size<Pass<T, true, true>>(*args) : cluster_size<Pass<T, true, false>>(*args);
    return backward ? cluster_size<Pass<T, false, true>>(*args) : cluster_size<Pass<T, false, false>>(*args);
  };
  return args->value.dtype == M3_F32 ? of(0.0f) : of(__half());
}

extern "C" int m3_gated_scan_fwd(const m3_gated_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_gated_args& a = *args;
  const int rc = check(a, false);
  if (rc != M3_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launched("gated scan", a.value.dtype == M3_BF16  ? launch_fwd<__nv_bfloat16>(a, s)
                                : a.value.dtype == M3_F16 ? launch_fwd<__half>(a, s)
                                                          : launch_fwd<float>(a, s));
}

extern "C" int m3_gated_scan_bwd(const m3_gated_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_gated_args& a = *args;
  const int rc = check(a, true);
  if (rc != M3_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return launched("gated scan backward", a.value.dtype == M3_BF16  ? launch_bwd<__nv_bfloat16>(a, s)
                                         : a.value.dtype == M3_F16 ? launch_bwd<__half>(a, s)
                                                                   : launch_bwd<float>(a, s));
}
