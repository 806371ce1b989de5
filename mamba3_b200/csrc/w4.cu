// Few-row projection with 4-bit weights: y[r][o] = sum_i x[r][i] s[o][g] (q[o][i] - z[o][g]), g = i / group.
//
// Codes are packed two to a byte, the even column in the low half, rows of (in_dim + 1) / 2 bytes;
// scales (and zero points, 8 where there are none) are one value per row and group.
//
// What bounds it is the stream of the codes, O I / 2 bytes, and their conversion on the way: at the copy rate an SM has
// about 2.7 instructions of a lane for a code, a conversion to float32 and a multiply-add take as many. So the
// products go to the warp-level tensor instruction (m16n8k16: 16 outputs x 8 rows of x), whose 16-bit operands take
// two codes at a time: bits of (1024 + code) less 1032 is code - 8 exactly (in bf16: 128 and 136). Which column goes
// where in a product is free as long as both operands agree, so the codes are used as they lie in memory: four
// threads share an output row, and of every group a thread has group / 4 neighbouring columns, one load of 4, 8 or
// 16 bytes. Products of 16-bit values by code - 8 are exact, sums float32, scaled group by group:
//   y = sum_g s (sum x (q - 8) - (z - 8) sum x),
// the sums of x by products with ones; y is rounded once.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "umma.cuh"

namespace m3 {

int report_error(int code, const char* msg);

namespace {

constexpr int kSlab = 128;  // columns that a warp takes at a time, 4 words of 8 codes a thread and output row
constexpr int kAhead = 2;   // slabs that are under way

// ---- codes ---------------------------------------------------------------------------------------

// Two codes to two values code - 8 in T: bytes 0 and 2 of v hold them in their low halves.
template <typename T> __device__ __forceinline__ uint32_t open2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t w = (v & 0x000F000Fu) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6408)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t w = (v & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 r =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// The 8 codes of a word, neighbours in pairs: byte b of v and of v >> 4 hold codes 2 b and 2 b + 1.
template <typename T> __device__ __forceinline__ void open8(uint32_t v, uint32_t (&pairs)[4]) {
  const uint32_t odd = v >> 4;
  pairs[0] = open2<T>(__byte_perm(v, odd, 0x0400));
  pairs[1] = open2<T>(__byte_perm(v, odd, 0x0501));
  pairs[2] = open2<T>(__byte_perm(v, odd, 0x0602));
  pairs[3] = open2<T>(__byte_perm(v, odd, 0x0703));
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// N words of one output row from byte `at` on; bytes past the row are 0 (x is 0 there). kAligned: whole words lie
// on multiples of their size; otherwise, and at the row's end, byte by byte.
template <bool kAligned, int N>
__device__ __forceinline__ void load_words(const uint8_t* row, int64_t at, int64_t bytes, int64_t stride, uint32_t* w) {
  if (kAligned && at + 4 * N <= bytes) {
    if constexpr (N == 1) {
      w[0] = __ldcs(reinterpret_cast<const unsigned int*>(row + at));
    } else if constexpr (N == 2) {
      const uint2 v = __ldcs(reinterpret_cast<const uint2*>(row + at));
      w[0] = v.x;
      w[1] = v.y;
    } else {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + at));
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (at + 4 * i + b < bytes) w[i] |= (uint32_t)row[(at + 4 * i + b) * stride] << (8 * b);
  }
}

// A warp's 16 output rows, as a thread sees them: rows g and g + 8 (past the end, the last one again: not written).
template <typename T, int kWords, bool kAligned> struct Weight {
  static constexpr int kGroup = 32 * kWords, kPerSlab = kSlab / kGroup;
  struct Slab {
    uint32_t code[2][4];
    float scale[2][kPerSlab], shift[2][kPerSlab];  // s and s (z - 8) of the slab's groups
  };
  const m3_w4_args& a;
  const uint8_t* code[2];
  int64_t scale_at[2], zero_at[2], bytes;
  int t;

  __device__ __forceinline__ Weight(const m3_w4_args& args, int64_t o0, int lane) : a(args), bytes((args.in_dim + 1) / 2), t(lane & 3) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t o = min(o0 + (lane >> 2) + 8 * r, a.out_dim - 1);
      code[r] = static_cast<const uint8_t*>(a.codes.data) + o * a.codes.stride[0];
      scale_at[r] = o * a.scales.stride[0];
      zero_at[r] = o * a.zeros.stride[0];
    }
  }
  // Pull a slab's codes towards L2.
  __device__ __forceinline__ void prefetch(int64_t slab) const {
    const int64_t at = slab * (kSlab / 2) + t * 16;
    if (at < bytes)
#pragma unroll
      for (int r = 0; r < 2; ++r) asm volatile("prefetch.global.L2 [%0];" ::"l"(code[r] + at * a.codes.stride[1]));
  }
  __device__ __forceinline__ void fetch(int64_t slab, Slab& to) const {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < kPerSlab; ++c) {
        load_words<kAligned, kWords>(code[r], slab * (kSlab / 2) + c * (kGroup / 2) + t * 4 * kWords, bytes, a.codes.stride[1],
                                     &to.code[r][c * kWords]);
        const int64_t group = slab * kPerSlab + c;
        const bool there = group * kGroup < a.in_dim;
        to.scale[r][c] = there ? ld_t(a.scales, scale_at[r] + group * a.scales.stride[1]) : 0.0f;
        to.shift[r][c] = there && a.zeros.data ? ld_t(a.zeros, zero_at[r] + group * a.zeros.stride[1]) - 8.0f : 0.0f;
      }
  }
};

// acc += scale (products - shift sums): the sums of one group, of a thread's 2 x 2 results.
__device__ __forceinline__ void join(float (&acc)[4], const float (&d)[4], const float (&sums)[4], const float s0, const float s1,
                                     const float z0, const float z1) {
  acc[0] = fmaf(s0, fmaf(-z0, sums[0], d[0]), acc[0]);
  acc[1] = fmaf(s0, fmaf(-z0, sums[1], d[1]), acc[1]);
  acc[2] = fmaf(s1, fmaf(-z1, sums[0], d[2]), acc[2]);
  acc[3] = fmaf(s1, fmaf(-z1, sums[1], d[3]), acc[3]);
}

// 8 columns of a row of x, from column c on; 0 past the row.
template <typename T>
__device__ __forceinline__ uint4 x_unit(const m3_w4_args& a, const T* row, int64_t c, bool units) {
  if (units && c + 8 <= a.in_dim) return *reinterpret_cast<const uint4*>(row + c);
  alignas(16) T w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = c + e < a.in_dim ? row[(c + e) * a.x.stride[1]] : from_f<T>(0.0f);
  return *reinterpret_cast<const uint4*>(w);
}

__device__ __forceinline__ bool x_in_units(const m3_w4_args& a) {
  return a.x.stride[1] == 1 && a.x.stride[0] % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x.data) & 15) == 0;
}

// ---- up to 8 rows --------------------------------------------------------------------------------
// A stream of codes: one CTA for 16 outputs, its warps share the columns out, slab by slab, and meet in shared memory.
// x, a few KB, comes from L1 as the products want it.
constexpr int kMostWarps = 16;

template <typename T, int kWords, bool kAligned>
__global__ void __launch_bounds__(32 * kMostWarps) w4_few_kernel(const m3_w4_args a) {
  using W = Weight<T, kWords, kAligned>;
  __shared__ float part[kMostWarps][8][16];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t o0 = (int64_t)blockIdx.x * 16, slabs = (a.in_dim + kSlab - 1) / kSlab;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const W weight(a, o0, lane);
  // Launched as a programmatic dependent: what the kernel before wrote, the weight too if it did, is there only after
  // the wait. Until then the first codes are pulled towards L2.
  for (int i = 0; i < kAhead; ++i) weight.prefetch(warp + i * warps);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool units = x_in_units(a), here = g < a.rows;
  const T* row = static_cast<const T*>(a.x.data) + g * a.x.stride[0];
  typename W::Slab held[kAhead];
  uint4 x[kAhead][4];
  auto fetch = [&](int64_t slab, typename W::Slab& w, uint4 (&u)[4]) {
    if (slab >= slabs) return;
    weight.fetch(slab, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // columns of word i of a thread: group i / kWords of the slab
      const int64_t c = slab * kSlab + i / kWords * W::kGroup + 8 * (kWords * t + i % kWords);
      u[i] = here ? x_unit(a, row, c, units) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(warp + i * warps, held[i], x[i]);
  const uint32_t one2 = std::is_same<T, __half>::value ? 0x3C003C00u : 0x3F803F80u;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t slab = warp; slab < slabs; slab += kAhead * warps) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (slab + i * warps >= slabs) break;
#pragma unroll
      for (int c = 0; c < W::kPerSlab; ++c) {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          uint32_t low[4], high[4];
          open8<T>(held[i].code[0][c * kWords + w], low);
          open8<T>(held[i].code[1][c * kWords + w], high);
          const uint4 b = x[i][c * kWords + w];
          mma<T>(d, low[0], high[0], low[1], high[1], b.x, b.y);
          mma<T>(d, low[2], high[2], low[3], high[3], b.z, b.w);
          if (a.zeros.data) {
            mma<T>(sums, one2, one2, one2, one2, b.x, b.y);
            mma<T>(sums, one2, one2, one2, one2, b.z, b.w);
          }
        }
        join(acc, d, sums, held[i].scale[0][c], held[i].scale[1][c], held[i].shift[0][c], held[i].shift[1][c]);
      }
      fetch(slab + (i + kAhead) * warps, held[i], x[i]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[warp][2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[e];
  __syncthreads();
  T* yp = static_cast<T*>(a.y.data);
  for (int i = threadIdx.x; i < 8 * 16; i += blockDim.x) {
    const int r = i >> 4;
    const int64_t out = o0 + (i & 15);
    if (r >= a.rows || out >= a.out_dim) continue;
    float v = 0.0f;
    for (int w = 0; w < warps; ++w) v += part[w][r][i & 15];
    yp[r * a.y.stride[0] + out * a.y.stride[1]] = from_f<T>(v);
  }
}

// ---- more rows -----------------------------------------------------------------------------------
// One CTA for 64 outputs and 8 kTiles rows of x: four warps of 16 outputs on even slabs, four on odd ones. x passes
// through a ring of panels of two slabs in shared memory, which the eight warps share: read by every CTA, it
// costs more than the codes.
constexpr int kManyThreads = 256, kPanel = 2 * kSlab, kPanels = 3;

// A panel's rows of 16-byte units (8 columns). A product reads a unit of each of 8 rows by four threads, group / 32
// units apart: the rows' pitch, and for groups of 128 a swap of units, spread them over all banks.
template <int kWords> constexpr int kPitch = kPanel + (kWords == 1 ? 32 : kWords == 2 ? 8 : 16);  // in 16-bit values
template <int kWords> __device__ __forceinline__ int unit_at(int u) { return kWords == 4 ? u ^ (u >> 3 & 1) : u; }

template <typename T, int kWords, bool kAligned, int kTiles>
__global__ void __launch_bounds__(kManyThreads) w4_many_kernel(const m3_w4_args a) {
  using W = Weight<T, kWords, kAligned>;
  constexpr int kRows = 8 * kTiles, kPit = kPitch<kWords>, kUnits = kPanel / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  T* xs = reinterpret_cast<T*>(smem);  // [kPanels][kRows][kPit]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, half = warp >> 2;
  const int64_t o0 = (int64_t)blockIdx.x * 64 + (warp & 3) * 16;
  const int64_t rows0 = (int64_t)blockIdx.y * kRows;
  const int rows = (int)min((int64_t)kRows, a.rows - rows0), tiles = (rows + 7) / 8;
  const int64_t slabs = (a.in_dim + kSlab - 1) / kSlab, panels = (slabs + 1) / 2;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const W weight(a, o0, lane);
  weight.prefetch(half);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool units = x_in_units(a);
  const T* xp = static_cast<const T*>(a.x.data) + rows0 * a.x.stride[0];
  auto stage = [&](int64_t panel) {
    if (panel < panels) {
      T* to = xs + panel % kPanels * kRows * kPit;
      for (int i = threadIdx.x; i < tiles * 8 * kUnits; i += kManyThreads) {
        const int r = i / kUnits, u = i % kUnits;
        const int64_t c = panel * kPanel + 8 * u;
        T* at = to + r * kPit + 8 * unit_at<kWords>(u);
        const T* row = xp + (r < rows ? r : 0) * a.x.stride[0];
        if (units && (c + 8 <= a.in_dim || c >= a.in_dim)) {
          const bool there = r < rows && c < a.in_dim;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(at))),
                       "l"(there ? row + c : row), "r"(there ? 16 : 0)
                       : "memory");
        } else {
          *reinterpret_cast<uint4*>(at) = r < rows ? x_unit(a, row, c, false) : make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < kPanels - 1; ++i) stage(i);
  typename W::Slab held[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (half + 2 * i < slabs) weight.fetch(half + 2 * i, held[i]);
  const uint32_t one2 = std::is_same<T, __half>::value ? 0x3C003C00u : 0x3F803F80u;
  float acc[kTiles][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.0f;
  for (int64_t panel0 = 0; panel0 < panels; panel0 += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t panel = panel0 + i, slab = 2 * panel + half;
      if (panel >= panels) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(kPanels - 2) : "memory");
      __syncthreads();  // this panel is there, and everyone is done with the one before
      stage(panel + kPanels - 1);
      if (slab < slabs) {
        const T* from = xs + panel % kPanels * kRows * kPit + g * kPit;
#pragma unroll
        for (int c = 0; c < W::kPerSlab; ++c) {
          uint32_t low[kWords][4], high[kWords][4];
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            open8<T>(held[i].code[0][c * kWords + w], low[w]);
            open8<T>(held[i].code[1][c * kWords + w], high[w]);
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            if (n >= tiles) break;
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              const uint4 b = *reinterpret_cast<const uint4*>(
                  from + 8 * n * kPit + 8 * unit_at<kWords>((half * W::kPerSlab + c) * 4 * kWords + t * kWords + w));
              mma<T>(d, low[w][0], high[w][0], low[w][1], high[w][1], b.x, b.y);
              mma<T>(d, low[w][2], high[w][2], low[w][3], high[w][3], b.z, b.w);
              if (a.zeros.data) {
                mma<T>(sums, one2, one2, one2, one2, b.x, b.y);
                mma<T>(sums, one2, one2, one2, one2, b.z, b.w);
              }
            }
            join(acc[n], d, sums, held[i].scale[0][c], held[i].scale[1][c], held[i].shift[0][c], held[i].shift[1][c]);
          }
        }
        if (slab + 2 * kAhead < slabs) weight.fetch(slab + 2 * kAhead, held[i]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);  // [4][kTiles][4][32]: the odd slabs' sums
  if (half == 1)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[(((warp & 3) * kTiles + n) * 4 + e) * 32 + lane] = acc[n][e];
  __syncthreads();
  if (half == 1) return;
  T* yp = static_cast<T*>(a.y.data);
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 8 * n + 2 * t + (e & 1);
      const int64_t out = o0 + g + 8 * (e >> 1);
      if (r < rows && out < a.out_dim)
        yp[(rows0 + r) * a.y.stride[0] + out * a.y.stride[1]] = from_f<T>(acc[n][e] + part[((warp * kTiles + n) * 4 + e) * 32 + lane]);
    }
}

// ---- host ----------------------------------------------------------------------------------------

cudaLaunchConfig_t config(dim3 grid, int threads, size_t smem, cudaStream_t stream, cudaLaunchAttribute* chained) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  chained->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  chained->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = chained;
  cfg.numAttrs = 1;
  return cfg;
}

template <typename T, int kWords, bool kAligned, int kTiles> cudaError_t launch_many(const m3_w4_args& a, cudaStream_t stream) {
  constexpr size_t smem = (size_t)kPanels * 8 * kTiles * kPitch<kWords> * 2;
  static_assert(smem >= 4 * kTiles * 4 * 32 * 4, "the odd slabs' sums fit the panels");
  auto kernel = w4_many_kernel<T, kWords, kAligned, kTiles>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute chained;
  const dim3 grid((unsigned)((a.out_dim + 63) / 64), (unsigned)((a.rows + 8 * kTiles - 1) / (8 * kTiles)));
  const cudaLaunchConfig_t cfg = config(grid, kManyThreads, smem, stream, &chained);
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int kWords, bool kAligned> cudaError_t launch_rows(const m3_w4_args& a, cudaStream_t stream) {
  if (a.rows <= 8) {
    // warps for the columns of 16 outputs: enough to give every SM 16, while each has two slabs or more
    const int64_t tiles = (a.out_dim + 15) / 16, slabs = (a.in_dim + kSlab - 1) / kSlab;
    int warps = 4;
    while (warps < kMostWarps && tiles * warps < (int64_t)16 * sm_count() && 4 * warps <= slabs) warps *= 2;
    cudaLaunchAttribute chained;
    const cudaLaunchConfig_t cfg = config(dim3((unsigned)tiles), 32 * warps, 0, stream, &chained);
    return cudaLaunchKernelEx(&cfg, w4_few_kernel<T, kWords, kAligned>, a);
  }
  if (a.rows <= 16) return launch_many<T, kWords, kAligned, 2>(a, stream);
  if (a.rows <= 32) return launch_many<T, kWords, kAligned, 4>(a, stream);
  return launch_many<T, kWords, kAligned, 8>(a, stream);  // past 64 rows, the weight is read once for every 64
}

template <typename T, int kWords> cudaError_t launch_group(const m3_w4_args& a, cudaStream_t stream) {
  const bool aligned = a.codes.stride[1] == 1 && a.codes.stride[0] % (4 * kWords) == 0 &&
                       reinterpret_cast<uintptr_t>(a.codes.data) % (4 * kWords) == 0;
  return aligned ? launch_rows<T, kWords, true>(a, stream) : launch_rows<T, kWords, false>(a, stream);
}

template <typename T> cudaError_t launch_type(const m3_w4_args& a, cudaStream_t stream) {
  switch (a.group) {
    case 32: return launch_group<T, 1>(a, stream);
    case 64: return launch_group<T, 2>(a, stream);
    default: return launch_group<T, 4>(a, stream);
  }
}

}  // namespace
}  // namespace m3

extern "C" int m3_linear_w4(const m3_w4_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_w4_args& a = *args;
  if (a.rows <= 0 || a.out_dim <= 0 || a.in_dim <= 0)
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: rows, out_dim and in_dim must be positive");
  if (a.rows > 64 * 65535 || a.out_dim > INT32_MAX || a.in_dim > INT32_MAX)
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: rows above 64 * 65535, or out_dim or in_dim above 2^31 - 1");
  if (a.group != 32 && a.group != 64 && a.group != 128)
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: group must be 32, 64 or 128");
  if (!a.x.data || !a.codes.data || !a.scales.data || !a.y.data)
    return report_error(M3_ERR_ARGUMENT, "m3_linear_w4: x, codes, scales and y are required");
  if ((a.x.dtype != M3_BF16 && a.x.dtype != M3_F16) || a.y.dtype != a.x.dtype || a.codes.dtype != M3_U8 ||
      a.scales.dtype < M3_F32 || a.scales.dtype > M3_BF16 || (a.zeros.data && a.zeros.dtype != a.scales.dtype))
    return report_error(M3_ERR_DTYPE, "m3_linear_w4: x and y share one 16-bit dtype, codes are bytes, scales and zeros "
                                      "share one float dtype");
  if (a.x.ndim != 2 || a.codes.ndim != 2 || a.scales.ndim != 2 || a.y.ndim != 2 || (a.zeros.data && a.zeros.ndim != 2))
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: every tensor has two dimensions");
  if (a.device >= 0 && cudaSetDevice(a.device) != cudaSuccess)
    return report_error(M3_ERR_CUDA, "m3_linear_w4: cannot select the device");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.x.dtype == M3_BF16 ? launch_type<__nv_bfloat16>(a, s) : launch_type<__half>(a, s);
  if (e != cudaSuccess)
    return report_error(M3_ERR_CUDA, (std::string("m3_linear_w4 launch failed: ") + cudaGetErrorString(e)).c_str());
  return M3_OK;
}
