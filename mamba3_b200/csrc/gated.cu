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
#include <string>

#include "common.cuh"
#include "umma.cuh"

namespace m3 {

int report_error(int code, const char* msg);

namespace {

constexpr int kTile = 64;      // tokens a tile: the training forward keeps the state before each
constexpr int kChannels = 64;  // channels a CTA
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRun = kTile / kWarps;  // consecutive tokens of a thread; it has two neighbouring channels
constexpr float kFloor = 1e-37f;      // least product of decays without a reset: see fold()

// f = sigmoid(x) and 1 - f = sigmoid(-x), both to a few units in the last place; x below -80 is taken as -80
// (f = 2e-35), so that exp stays finite; NaN stays NaN.
__device__ __forceinline__ void keep_lose(float x, float& keep, float& lose) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(x), "f"(-80.0f));
  const float e = __expf(-c);
  keep = __fdividef(1.0f, 1.0f + e);
  lose = e * keep;
}

__device__ __forceinline__ float sigmoid_approx(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// A run of tokens as a map of the state before it: h -> a h + h0. a is exactly 0 where a reset lies in the run,
// and then nothing of h passes, not even an infinity or NaN; otherwise a product of decays is kept at kFloor or
// more, so that an infinity or NaN before the run does pass.
__device__ __forceinline__ float fold(float a, float h0, float h) { return a == 0.0f ? h0 : fmaf(a, h, h0); }

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

// ---- tiles ---------------------------------------------------------------------------------------

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Start copying tokens t0 .. t0 + 63 of channels c0 .. c0 + 63 to a tile [64][64]; what is outside reads as 0.
template <typename T, bool kVec>
__device__ __forceinline__ void load_tile(T* tile, const m3_tensor& from, int b, int64_t t0, int c0, int64_t length, int channels) {
  const T* base = static_cast<const T*>(from.data) + b * from.stride[0];
  if constexpr (kVec) {  // 16-byte words of a token's channels, each inside or outside as a whole
    constexpr int kWord = 16 / sizeof(T), kRow = kChannels / kWord;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(tile));
#pragma unroll
    for (int i = threadIdx.x; i < kTile * kRow; i += kThreads) {
      const int t = i / kRow, c = i % kRow * kWord;
      const bool there = t0 + t < length && c0 + c < channels;
      copy16(to + (t * kChannels + c) * sizeof(T), there ? base + (t0 + t) * from.stride[1] + c0 + c : base, there);
    }
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < kTile * kChannels; i += kThreads) {
      const int t = i / kChannels, c = i % kChannels;
      tile[i] = t0 + t < length && c0 + c < channels ? base[(t0 + t) * from.stride[1] + (c0 + c) * from.stride[2]]
                                                      : from_f<T>(0.0f);
    }
  }
}

template <typename T> __device__ __forceinline__ float2 read_two(const T* tile, int token, int lane) {
  return Two<T>::open(reinterpret_cast<const typename Two<T>::word*>(tile + token * kChannels)[lane]);
}

template <typename T, bool kVec>
__device__ __forceinline__ void write_two(const m3_tensor& to, int64_t at, int c, int channels, float2 v) {
  T* p = static_cast<T*>(to.data) + at;
  if constexpr (kVec) {
    if (c < channels) *reinterpret_cast<typename Two<T>::word*>(p + c) = Two<T>::close(v);
  } else {
    if (c < channels) p[c * to.stride[2]] = from_f<T>(v.x);
    if (c + 1 < channels) p[(c + 1) * to.stride[2]] = from_f<T>(v.y);
  }
}

// Bits 0 .. kRun - 1: which tokens of this warp's run are resets. Read by the first lanes, a tile ahead.
__device__ __forceinline__ bool read_reset(const m3_tensor& reset, int b, int64_t t, int64_t length, int lane) {
  return reset.data && lane < kRun && t + lane < length &&
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
__device__ __forceinline__ void store_in(int rank, float4* local, float4 v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(local))), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

constexpr int kMaxCluster = 16;

// Shared memory of a CTA: kStages buffers of its tensors' tiles, the maps of its warps' runs (float4 = a, a', h0, h0'
// of a lane's two channels; the backward's second array has the reverse maps' h0, h0'), and in clusters the maps of
// the cluster's tiles, for even and odd groups of tiles.
constexpr int kStages = 2;
template <typename T> __host__ __device__ constexpr int tile_bytes() { return kTile * kChannels * (int)sizeof(T); }
constexpr int kRunMaps = kWarps * 32 * 16;
__host__ __device__ constexpr int smem_bytes(int tile_bytes, int tensors, int run_maps, int cluster) {
  return kStages * tensors * tile_bytes + run_maps * kRunMaps + (cluster > 1 ? 2 * cluster * 32 * 16 : 0);
}

// Leave `map`, of this CTA's tile, in every CTA of the cluster, and wait for theirs: maps[rank][lane].
__device__ __forceinline__ void exchange(float4* maps, int rank, int cluster, int warp, int lane, float4 map) {
  if (warp == 0)
    for (int r = 0; r < cluster; ++r) store_in(r, maps + rank * 32 + lane, map);
  __syncwarp();
  cluster_arrive();
  cluster_wait();
}

// The map of one run after another.
__device__ __forceinline__ void join(float4& m, float4 next) {
  m.z = fold(next.x, next.z, m.z);
  m.w = fold(next.y, next.w, m.w);
  m.x = m.x == 0.0f || next.x == 0.0f ? 0.0f : fmaxf(m.x * next.x, kFloor);
  m.y = m.y == 0.0f || next.y == 0.0f ? 0.0f : fmaxf(m.y * next.y, kFloor);
}

// Forward. One pass over the inputs: a thread folds its run of 8 tokens into a map (a, h0), the maps of the 8 runs
// of a tile (and of a cluster's tiles) give every run the state before it, and the run is repeated from there
// out of registers. CTAs walk a sequence's tiles one after another; where sequences and channels are too few to
// fill the GPU, a cluster walks them together.
template <typename T, bool kGate, bool kVec>
__global__ void __launch_bounds__(kThreads, 3) gated_fwd_kernel(const m3_gated_args a, int cluster) {
  constexpr int kTensors = kGate ? 3 : 2, kElems = kTile * kChannels;
  extern __shared__ __align__(16) uint8_t smem[];
  T* tiles = reinterpret_cast<T*>(smem);
  float4* runs = reinterpret_cast<float4*>(smem + kStages * kTensors * tile_bytes<T>());
  float4* peers = runs + kWarps * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? cluster_rank() : 0;
  const int b = blockIdx.y, c0 = blockIdx.x / cluster * kChannels, c = c0 + 2 * lane;
  const int64_t ntiles = (a.length + kTile - 1) / kTile, groups = (ntiles + cluster - 1) / cluster;
  auto load = [&](int64_t g) {
    const int64_t t = g * cluster + rank;
    if (g < groups && t < ntiles) {
      T* to = tiles + (g % kStages) * kTensors * kElems;
      load_tile<T, kVec>(to, a.forget, b, t * kTile, c0, a.length, a.channels);
      load_tile<T, kVec>(to + kElems, a.value, b, t * kTile, c0, a.length, a.channels);
      if constexpr (kGate) load_tile<T, kVec>(to + 2 * kElems, a.gate, b, t * kTile, c0, a.length, a.channels);
    }
    copies_commit();
  };
  float2 carry = read_state(a.state, b, c, a.channels);  // the state before the group of tiles
  for (int g = 0; g < kStages - 1; ++g) load(g);
  bool flag = read_reset(a.reset, b, (int64_t)rank * kTile + warp * kRun, a.length, lane);
  if (cluster > 1) {  // the others have started: their shared memory may be written
    cluster_arrive();
    cluster_wait();
  }
  for (int64_t g = 0; g < groups; ++g) {
    const int64_t t = g * cluster + rank, t0 = t * kTile + warp * kRun;
    const uint32_t resets = __ballot_sync(0xffffffffu, flag);
    flag = read_reset(a.reset, b, t0 + (int64_t)cluster * kTile, a.length, lane);
    copies_wait<kStages - 2>();
    __syncthreads();  // this group's tile is there, and everyone is done with the one before
    load(g + kStages - 1);
    const T* tile = tiles + (g % kStages) * kTensors * kElems;
    const int n = t0 >= a.length ? 0 : a.length - t0 < kRun ? (int)(a.length - t0) : kRun;  // tokens of this run
    float2 keep[kRun], in[kRun];
    float4 map = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
    float least = kFloor;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      keep[j] = make_float2(1.0f, 1.0f);
      in[j] = make_float2(0.0f, 0.0f);
      if (j < n) {
        const float2 f = read_two(tile, warp * kRun + j, lane), v = read_two(tile + kElems, warp * kRun + j, lane);
        float2 lose;
        keep_lose(f.x, keep[j].x, lose.x);
        keep_lose(f.y, keep[j].y, lose.y);
        in[j] = make_float2(lose.x * v.x, lose.y * v.y);
        if (resets >> j & 1u) map = make_float4(least = 0.0f, 0.0f, 0.0f, 0.0f);
        map.z = fmaf(keep[j].x, map.z, in[j].x);
        map.w = fmaf(keep[j].y, map.w, in[j].y);
        map.x = fmaxf(map.x * keep[j].x, least);
        map.y = fmaxf(map.y * keep[j].y, least);
      }
    }
    runs[warp * 32 + lane] = map;
    __syncthreads();
    float2 h = carry;  // the state before this CTA's tile
    if (cluster > 1) {
      float4 whole = runs[lane];
      if (warp == 0)
        for (int w = 1; w < kWarps; ++w) join(whole, runs[w * 32 + lane]);
      float4* maps = peers + (g & 1) * cluster * 32;
      exchange(maps, rank, cluster, warp, lane, whole);
      for (int r = 0; r < cluster; ++r) {
        if (r == rank) h = carry;
        const float4 m = maps[r * 32 + lane];
        carry.x = fold(m.x, m.z, carry.x);
        carry.y = fold(m.y, m.w, carry.y);
      }
    }
    if (a.carry.data && warp == 0 && t < ntiles) {
      float* to = static_cast<float*>(a.carry.data) + b * a.carry.stride[0] + t * a.carry.stride[1];
      if (c < a.channels) to[c] = h.x;
      if (c + 1 < a.channels) to[c + 1] = h.y;
    }
    const int upto = cluster > 1 ? warp : kWarps;  // alone, the state after the tile is the next one's
    float2 mine = h;
    for (int w = 0; w < upto; ++w) {
      if (w == warp) mine = h;
      const float4 m = runs[w * 32 + lane];
      h.x = fold(m.x, m.z, h.x);
      h.y = fold(m.y, m.w, h.y);
    }
    if (cluster > 1) mine = h;
    else carry = h;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (j >= n) break;
      if (resets >> j & 1u) mine = make_float2(0.0f, 0.0f);
      mine.x = fmaf(keep[j].x, mine.x, in[j].x);
      mine.y = fmaf(keep[j].y, mine.y, in[j].y);
      float2 y = mine;
      if constexpr (kGate) {
        const float2 q = read_two(tile + 2 * kElems, warp * kRun + j, lane);
        y.x *= q.x * sigmoid_approx(q.x);
        y.y *= q.y * sigmoid_approx(q.y);
      }
      write_two<T, kVec>(a.y, b * a.y.stride[0] + (t0 + j) * a.y.stride[1], c, a.channels, y);
    }
  }
  if (rank == 0 && warp == 0) write_state(a.out_state, b, c, a.channels, carry);
}

// Backward, the tiles from the last to the first: the states of a tile come from the state kept before it, as in
// the forward, and the gradients In run back through the same maps' a with h0 of their own.
template <typename T, bool kGate, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) gated_bwd_kernel(const m3_gated_args a, int cluster) {
  constexpr int kTensors = kGate ? 4 : 3, kElems = kTile * kChannels;
  extern __shared__ __align__(16) uint8_t smem[];
  T* tiles = reinterpret_cast<T*>(smem);
  float4* runs = reinterpret_cast<float4*>(smem + kStages * kTensors * tile_bytes<T>());
  float4* back = runs + kWarps * 32;  // (a, a', In0, In0') of the runs from the back
  float4* peers = back + kWarps * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? cluster_rank() : 0;
  const int b = blockIdx.y, c0 = blockIdx.x / cluster * kChannels, c = c0 + 2 * lane;
  const int64_t ntiles = (a.length + kTile - 1) / kTile, groups = (ntiles + cluster - 1) / cluster;
  auto load = [&](int64_t g) {  // groups from the last, groups - 1, to 0
    const int64_t t = g * cluster + rank;
    if (g >= 0 && t < ntiles) {
      T* to = tiles + (g % kStages) * kTensors * kElems;
      load_tile<T, kVec>(to, a.forget, b, t * kTile, c0, a.length, a.channels);
      load_tile<T, kVec>(to + kElems, a.value, b, t * kTile, c0, a.length, a.channels);
      load_tile<T, kVec>(to + 2 * kElems, a.dy, b, t * kTile, c0, a.length, a.channels);
      if constexpr (kGate) load_tile<T, kVec>(to + 3 * kElems, a.gate, b, t * kTile, c0, a.length, a.channels);
    }
    copies_commit();
  };
  auto before = [&](int64_t t) {  // the state kept before tile t
    float2 h = make_float2(0.0f, 0.0f);
    if (t >= 0 && t < ntiles) {
      const float* from = static_cast<const float*>(a.carry.data) + b * a.carry.stride[0] + t * a.carry.stride[1];
      if (c < a.channels) h.x = from[c];
      if (c + 1 < a.channels) h.y = from[c + 1];
    }
    return h;
  };
  float2 carry = read_state(a.dstate, b, c, a.channels);  // In after the group of tiles
  for (int i = 0; i < kStages - 1; ++i) load(groups - 1 - i);
  bool flag = read_reset(a.reset, b, ((groups - 1) * cluster + rank) * kTile + warp * kRun, a.length, lane);
  float2 kept = before((groups - 1) * cluster + rank);
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
  }
  for (int64_t g = groups - 1; g >= 0; --g) {
    const int64_t t = g * cluster + rank, t0 = t * kTile + warp * kRun;
    const uint32_t resets = __ballot_sync(0xffffffffu, flag);
    float2 h = kept;
    if (g > 0) {
      flag = read_reset(a.reset, b, t0 - (int64_t)cluster * kTile, a.length, lane);
      kept = before(t - cluster);
    }
    copies_wait<kStages - 2>();
    __syncthreads();
    load(g - (kStages - 1));
    const T* tile = tiles + (g % kStages) * kTensors * kElems;
    const int n = t0 >= a.length ? 0 : a.length - t0 < kRun ? (int)(a.length - t0) : kRun;
    float2 keep[kRun], lose[kRun], dh[kRun];
    float4 map = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
    float least = kFloor;
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      keep[j] = make_float2(1.0f, 1.0f);
      lose[j] = dh[j] = make_float2(0.0f, 0.0f);
      if (j < n) {
        const int token = warp * kRun + j;
        const float2 f = read_two(tile, token, lane), v = read_two(tile + kElems, token, lane);
        keep_lose(f.x, keep[j].x, lose[j].x);
        keep_lose(f.y, keep[j].y, lose[j].y);
        dh[j] = read_two(tile + 2 * kElems, token, lane);
        if constexpr (kGate) {
          const float2 q = read_two(tile + 3 * kElems, token, lane);
          dh[j].x *= q.x * sigmoid_approx(q.x);
          dh[j].y *= q.y * sigmoid_approx(q.y);
        }
        if (resets >> j & 1u) map = make_float4(least = 0.0f, 0.0f, 0.0f, 0.0f);
        map.z = fmaf(keep[j].x, map.z, lose[j].x * v.x);
        map.w = fmaf(keep[j].y, map.w, lose[j].y * v.y);
        map.x = fmaxf(map.x * keep[j].x, least);
        map.y = fmaxf(map.y * keep[j].y, least);
      }
    }
    float4 rmap = make_float4(map.x, map.y, 0.0f, 0.0f);
#pragma unroll
    for (int j = kRun - 1; j >= 0; --j) {
      const bool cut = resets >> j & 1u;
      rmap.z = cut ? 0.0f : keep[j].x * (dh[j].x + rmap.z);
      rmap.w = cut ? 0.0f : keep[j].y * (dh[j].y + rmap.w);
    }
    runs[warp * 32 + lane] = map;
    back[warp * 32 + lane] = rmap;
    __syncthreads();
    float2 in = carry;  // In after this CTA's tile
    if (cluster > 1) {
      float4 whole = back[(kWarps - 1) * 32 + lane];
      if (warp == 0)
        for (int w = kWarps - 2; w >= 0; --w) join(whole, back[w * 32 + lane]);
      float4* maps = peers + (g & 1) * cluster * 32;
      exchange(maps, rank, cluster, warp, lane, whole);
      for (int r = cluster - 1; r >= 0; --r) {
        if (r == rank) in = carry;
        const float4 m = maps[r * 32 + lane];
        carry.x = fold(m.x, m.z, carry.x);
        carry.y = fold(m.y, m.w, carry.y);
      }
    }
    for (int w = 0; w < warp; ++w) {
      const float4 m = runs[w * 32 + lane];
      h.x = fold(m.x, m.z, h.x);
      h.y = fold(m.y, m.w, h.y);
    }
    const int downto = cluster > 1 ? warp + 1 : 0;
    float2 mine = in;
    for (int w = kWarps - 1; w >= downto; --w) {
      if (w == warp) mine = in;
      const float4 m = back[w * 32 + lane];
      in.x = fold(m.x, m.z, in.x);
      in.y = fold(m.y, m.w, in.y);
    }
    if (cluster > 1) mine = in;
    else carry = in;
    float2 prev[kRun];  // h_{t-1} as token t sees it
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      if (resets >> j & 1u) h = make_float2(0.0f, 0.0f);
      prev[j] = h;
      const float2 v = j < n ? read_two(tile + kElems, warp * kRun + j, lane) : make_float2(0.0f, 0.0f);
      h.x = fmaf(keep[j].x, h.x, lose[j].x * v.x);
      h.y = fmaf(keep[j].y, h.y, lose[j].y * v.y);
    }
#pragma unroll
    for (int j = kRun - 1; j >= 0; --j) {
      if (j >= n) continue;
      const int token = warp * kRun + j;
      const float2 v = read_two(tile + kElems, token, lane);
      if constexpr (kGate) {
        const float2 q = read_two(tile + 3 * kElems, token, lane), dy = read_two(tile + 2 * kElems, token, lane);
        const float2 s = make_float2(sigmoid_approx(q.x), sigmoid_approx(q.y));
        const float2 ht = make_float2(fmaf(keep[j].x, prev[j].x, lose[j].x * v.x), fmaf(keep[j].y, prev[j].y, lose[j].y * v.y));
        write_two<T, kVec>(a.dgate, b * a.dgate.stride[0] + (t0 + j) * a.dgate.stride[1], c, a.channels,
                           make_float2(dy.x * ht.x * (s.x * fmaf(q.x, 1.0f - s.x, 1.0f)),
                                       dy.y * ht.y * (s.y * fmaf(q.y, 1.0f - s.y, 1.0f))));
      }
      const float2 G = make_float2(dh[j].x + mine.x, dh[j].y + mine.y);
      write_two<T, kVec>(a.dvalue, b * a.dvalue.stride[0] + (t0 + j) * a.dvalue.stride[1], c, a.channels,
                         make_float2(G.x * lose[j].x, G.y * lose[j].y));
      write_two<T, kVec>(a.dforget, b * a.dforget.stride[0] + (t0 + j) * a.dforget.stride[1], c, a.channels,
                         make_float2(G.x * (prev[j].x - v.x) * (keep[j].x * lose[j].x),
                                     G.y * (prev[j].y - v.y) * (keep[j].y * lose[j].y)));
      const bool cut = resets >> j & 1u;
      mine.x = cut ? 0.0f : keep[j].x * G.x;
      mine.y = cut ? 0.0f : keep[j].y * G.y;
    }
  }
  if (a.dinitial.data && rank == 0 && warp == 0) write_state(a.dinitial, b, c, a.channels, carry);
}

// One token: nothing but elementwise work, one thread for kWide neighbouring channels.
template <typename T, int kWide>
__global__ void __launch_bounds__(128) gated_step_kernel(const m3_gated_args a) {
  const int c = (blockIdx.x * 128 + threadIdx.x) * kWide, b = blockIdx.y;
  if (c >= a.channels) return;
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
    keep_lose(f[e], keep, lose);
    h[e] = fmaf(keep, reset ? 0.0f : h[e], lose * v[e]);
    y[e] = a.gate.data ? h[e] * (q[e] * sigmoid_approx(q[e])) : h[e];
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
  const dim3 grid((unsigned)((a.channels + per_block - 1) / per_block), (unsigned)a.batch);
  if (wide) gated_step_kernel<T, 4><<<grid, 128, 0, stream>>>(a);
  else gated_step_kernel<T, 1><<<grid, 128, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename K> cudaError_t launch_tiles(K kernel, const m3_gated_args& a, int tile, int tensors, int run_maps, cudaStream_t stream) {
  const int64_t ntiles = (a.length + kTile - 1) / kTile;
  const int64_t blocks = (int64_t)a.batch * ((a.channels + kChannels - 1) / kChannels);
  // CTAs that fit the GPU: a cluster takes a sequence's tiles together while its CTAs still have room at once
  // (past 8 CTAs, a cluster's size without conditions, only where two fit an SM)
  const int per_sm = 227 * 1024 / (smem_bytes(tile, tensors, run_maps, 2) + 1024);
  const int64_t room = (int64_t)sm_count() * per_sm;
  const int most = per_sm > 1 ? kMaxCluster : 8;
  int cluster = 1;
  while (cluster < most && 2 * cluster <= ntiles && 2 * cluster * blocks <= room) cluster *= 2;
  const int smem = smem_bytes(tile, tensors, run_maps, cluster);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (cluster > 8) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.channels + kChannels - 1) / kChannels * cluster), (unsigned)a.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, a, cluster);
}

template <typename T> cudaError_t launch_fwd(const m3_gated_args& a, cudaStream_t stream) {
  if (a.length == 1) return launch_step_token<T>(a, stream);
  constexpr int kElem = sizeof(T), kWord = 16 / kElem;
  const bool vec = a.channels % kWord == 0 && rows_aligned(a.value, kElem, 16) && rows_aligned(a.forget, kElem, 16) &&
                   rows_aligned(a.gate, kElem, 16) && rows_aligned(a.y, kElem, 2 * kElem);
  constexpr int tile = tile_bytes<T>();
  if (a.gate.data)
    return vec ? launch_tiles(gated_fwd_kernel<T, true, true>, a, tile, 3, 1, stream)
               : launch_tiles(gated_fwd_kernel<T, true, false>, a, tile, 3, 1, stream);
  return vec ? launch_tiles(gated_fwd_kernel<T, false, true>, a, tile, 2, 1, stream)
             : launch_tiles(gated_fwd_kernel<T, false, false>, a, tile, 2, 1, stream);
}

template <typename T> cudaError_t launch_bwd(const m3_gated_args& a, cudaStream_t stream) {
  constexpr int kElem = sizeof(T), kWord = 16 / kElem;
  const bool vec = a.channels % kWord == 0 && rows_aligned(a.value, kElem, 16) && rows_aligned(a.forget, kElem, 16) &&
                   rows_aligned(a.gate, kElem, 16) && rows_aligned(a.dy, kElem, 16) && rows_aligned(a.dvalue, kElem, 2 * kElem) &&
                   rows_aligned(a.dforget, kElem, 2 * kElem) && rows_aligned(a.dgate, kElem, 2 * kElem);
  constexpr int tile = tile_bytes<T>();
  if (a.gate.data)
    return vec ? launch_tiles(gated_bwd_kernel<T, true, true>, a, tile, 4, 2, stream)
               : launch_tiles(gated_bwd_kernel<T, true, false>, a, tile, 4, 2, stream);
  return vec ? launch_tiles(gated_bwd_kernel<T, false, true>, a, tile, 3, 2, stream)
             : launch_tiles(gated_bwd_kernel<T, false, false>, a, tile, 3, 2, stream);
}

bool shaped(const m3_tensor& t, int ndim, int dtype) { return t.data == nullptr || (t.ndim == ndim && t.dtype == dtype); }

int check(const m3_gated_args& a, bool backward) {
  if (a.batch <= 0 || a.length <= 0 || a.channels <= 0)
    return report_error(M3_ERR_SHAPE, "gated scan: batch, length and channels must be positive");
  if (a.batch > 65535) return report_error(M3_ERR_SHAPE, "gated scan: batch above 65535");
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
