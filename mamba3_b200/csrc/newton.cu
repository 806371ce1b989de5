// Newton-Schulz orthogonalisation of optimiser updates, a stack of [rows, cols] matrices.
//
// X_0 = G / |G|_F (0 for G = 0), m <= n after a transposition where rows > cols, then `steps` times
//   A = X X^T,   P = b A + c A A,   X <- a X + P X.
// Each line is one launch of a tcgen05 product kernel: fp16 operands staged by TMA, float32
// accumulators in tensor memory, the sums of the formula in the epilogue.
//
// Rounding. The operands are float16, not bfloat16: with 8 significand bits the five steps leave the
// result 1 to 2 % off, with 11 bits 0.1 %. Entries are held times 256 (X, A and P have entries of at
// most a few units, and typical ones of 1e-4 to 1e-6, which float16 would hold as subnormals); 256 leaves
// room up to 255 before infinity. P's diagonal is kept apart in float32 and joins a in the epilogue,
// X <- (a + P_ii) X + (P - diag) X: near the fixed point a = 3.44 and P_ii = -2.7 almost cancel, and a
// rounding of P_ii would count fivefold (0.13 % instead of 0.08 % of the result, 0.3 % for a vector).
// A rounding of X in the first steps is amplified by up to a = 3.44 a
// step in the directions of small singular values, so X_0 and X_1 also keep what their rounding dropped
// (`lo`), which the a X term adds back: a matrix with a few directions far above its noise
// comes out 5 times nearer (5e-4 against 2.7e-3 of its norm); later steps gain nothing from it.
// The squared norm is summed in float64 (a float32 sum of squares overflows above 2e19).
#include <algorithm>
#include <string>

#include "common.cuh"
#include "umma.cuh"

namespace m3 {

int report_error(int code, const char* msg);

// The error word of this unit's bounded waits, for m3_device_error(); the device is synchronised.
int read_newton_error(int clear) { return read_unit_error(clear); }

namespace newton {

using namespace umma;

constexpr float kHold = 256.0f;   // stored entries are the matrix's times this
constexpr int kNormParts = 296;   // partial sums of squares per matrix
constexpr int kNormThreads = 512;
constexpr int kLoSteps = 2;       // X_0 .. X_{kLoSteps - 1} keep their rounding residue

__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- the norm and X_0 ----------------------------------------------------------------------------

// 8 consecutive elements at `at` (16-byte aligned for 16-bit types, 32-byte for float32) to float.
__device__ __forceinline__ void load8(const m3_tensor& t, int64_t at, float* v) {
  if (t.dtype == M3_F32) {
    const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(t.data) + at);
    *reinterpret_cast<float4*>(v) = from[0];
    *reinterpret_cast<float4*>(v + 4) = from[1];
    return;
  }
  const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __half*>(t.data) + at);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = t.dtype == M3_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&words[e]))
                                       : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&words[e]));
    v[2 * e] = f.x;
    v[2 * e + 1] = f.y;
  }
}

// Sums of squares of one matrix, as rows of `cols` elements of stride col_stride. With `vec` the rows
// are runs of 8 aligned elements.
__global__ void __launch_bounds__(kNormThreads) norm_kernel(const m3_orth_args a, int64_t rows, int64_t cols, int64_t row_stride,
                                                            int64_t col_stride, bool vec, double* parts) {
  __shared__ double warp_part[kNormThreads / 32];
  dependents_may_start();
  const int64_t base = (int64_t)blockIdx.y * a.update.stride[0];
  const int64_t first = (int64_t)blockIdx.x * kNormThreads + threadIdx.x, step = (int64_t)kNormParts * kNormThreads;
  double ss = 0.0;
  if (vec) {
    const int64_t runs = cols / 8, total = rows * runs;
    for (int64_t i = first; i < total; i += 4 * step) {
      float v[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t j = i + u * step;
        if (j < total) {
          load8(a.update, base + (rows == 1 ? j * 8 : j / runs * row_stride + j % runs * 8), v[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u][e] = 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fma((double)v[u][e], (double)v[u][e], ss);
    }
  } else {
#pragma unroll 4
    for (int64_t i = first; i < rows * cols; i += step) {
      const double v = ld_t(a.update, base + i / cols * row_stride + i % cols * col_stride);
      ss = fma(v, v, ss);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kNormThreads / 32; ++w) t += warp_part[w];
    parts[(int64_t)blockIdx.y * kNormParts + blockIdx.x] = t;
  }
}

// hi + lo = 256 G / |G| as [m][ld], tiles of 64 x 64 through shared memory: the reads run along
// the dimension of G whose stride is 1, the writes along X's rows.
__global__ void __launch_bounds__(256) start_kernel(const m3_orth_args a, const double* parts, int m, int n, int64_t ld,
                                                    int64_t row_stride, int64_t col_stride, bool vec, __half* hi,
                                                    __half* lo) {
  __shared__ float tile[64][65];
  __shared__ float factor[2];
  const int tid = threadIdx.x;
  dependents_may_start();
  wait_for_previous();
  if (tid < 32) {
    double ss = 0.0;
    for (int p = tid; p < kNormParts; p += 32) ss += parts[(int64_t)blockIdx.y * kNormParts + p];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (tid == 0) {
      // two float32 factors whose product is 256 / |G|, which alone can be past float32's range
      const double inv = ss == 0.0 ? 0.0 : kHold / sqrt(ss);
      const double first = inv > 0.0 && inv < 1e300 ? scalbn(1.0, ilogb(inv) / 2) : 1.0;
      factor[0] = (float)first;
      factor[1] = (float)(inv / first);
    }
  }
  const int64_t base = (int64_t)blockIdx.y * a.update.stride[0];
  const bool along_rows = col_stride != 1;  // G's unit stride runs down X's columns
  const int across = (n + 63) / 64, tiles = across * ((m + 63) / 64);
  __syncthreads();
  const float f0 = factor[0], f1 = factor[1];
  for (int at = blockIdx.x; at < tiles; at += gridDim.x) {
    const int r0 = at / across * 64, c0 = at % across * 64;
    if (vec) {  // runs of 8 aligned elements along the unit stride, inside the matrix or outside as a whole
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = tid + 256 * u, along = (i & 7) * 8, other = i >> 3;
        const int r = along_rows ? along : other, c = along_rows ? other : along;
        float v[8] = {};
        if (r0 + r < m && c0 + c < n) load8(a.update, base + (r0 + r) * row_stride + (c0 + c) * col_stride, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[along_rows ? r + e : r][along_rows ? c : c + e] = v[e];
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < 64 * 64; i += 256) {
        const int r = along_rows ? i & 63 : i >> 6, c = along_rows ? i >> 6 : i & 63;
        tile[r][c] = r0 + r < m && c0 + c < n ? ld_t(a.update, base + (r0 + r) * row_stride + (c0 + c) * col_stride) : 0.0f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = tid + 256 * u, r = i >> 3, c = (i & 7) * 8;
      if (r0 + r >= m) continue;
      alignas(16) __half h[8], l[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = tile[r][c + e] * f0 * f1;
        h[e] = __float2half_rn(v);
        l[e] = __float2half_rn(v - __half2float(h[e]));
      }
      // ld is a multiple of 64: the columns past n are there
      const int64_t to = ((int64_t)blockIdx.y * m + r0 + r) * ld + c0 + c;
      *reinterpret_cast<uint4*>(hi + to) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(lo + to) = *reinterpret_cast<const uint4*>(l);
    }
    __syncthreads();
  }
}

// out = (hi + lo) / 256: the result of 0 steps.
__global__ void __launch_bounds__(256) finish_kernel(const m3_orth_args a, const __half* hi, const __half* lo, int m, int n,
                                                     int64_t ld, int64_t row_stride, int64_t col_stride) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)m * n) return;
  const int64_t r = i / n, c = i % n, at = ((int64_t)blockIdx.y * m + r) * ld + c;
  st_t(a.out, blockIdx.y * a.out.stride[0] + r * row_stride + c * col_stride,
       (__half2float(hi[at]) + __half2float(lo[at])) * (1.0f / kHold));
}

// ---- the product kernel --------------------------------------------------------------------------

// out = alpha L R + beta add over a stack of matrices; L [m][k], R [k][n].
struct Product {
  int m, n, k, tiles_m, tiles_n, tiles;  // tiles: of the whole stack
  int symmetric;                         // the product is: only tiles that reach the diagonal or lie above it
  float alpha, beta;
  int64_t ld;                            // row stride of add, out and their residues (a multiple of 64; the columns
                                         // past n are there); matrices m * ld apart
  const __half *add, *add_lo;            // null: no such term
  const float* add_diagonal;             // [matrix][m], joins beta row by row; null: none
  float* diagonal;                       // [matrix][m]: the diagonal goes there and out has 0 instead; null: it stays
  __half *out, *out_lo;                  // out null: the product, divided by 256, goes to `result`
  m3_tensor result;                      // strides (matrix, row, column) of X's orientation
};

constexpr int kTileM = 128, kTileK = 64;  // rows of a CTA's part of a tile; k a stage
constexpr uint32_t kBox = 2048;           // bytes of an epilogue box of 32 x 32 16-bit values

// A tile of 128 x BN a CTA, or (kPair) of 256 x BN a pair of CTAs, in which each loads its 128 rows of L
// and its half of R's columns and the pair's MMA reads both halves.
template <int BN, bool kPair> struct Shape {
  static constexpr int kRows = kPair ? 2 * kTileM : kTileM;
  static constexpr int kRight = kPair ? BN / 2 : BN;  // columns of R that a CTA loads
  static constexpr uint32_t kA = kTileM * kTileK * 2, kB = kRight * kTileK * 2;
  static constexpr int kStages = 196608 / (kA + kB);      // 6 or 8 stages of 32 or 24 KB
  // Epilogue warps: each takes a quarter of TMEM's lanes and a quarter (BN = 64: a half) of the columns.
  static constexpr int kWarps = BN == 64 ? 8 : 16, kBlocks = BN / 32 / (kWarps / 4);
  static constexpr int kThreads = 32 * (2 + kWarps);  // warp 0 loads, warp 1 issues the MMAs
  static constexpr uint32_t kBoxes = kStages * (kA + kB);  // a box for each of them
  static constexpr uint32_t kBars = kBoxes + kWarps * kBox;
  static constexpr uint32_t kBytes = kBars + 256 + 1024;  // + alignment slack
  static constexpr uint32_t kColumns = 2 * BN;            // two accumulators
};

struct Where {
  int matrix, i, j;  // which matrix of the stack, tile row, tile column
};

// Tile rows (of bm) of tile column j (of bn) that a symmetric product needs: those with an element on
// or above the diagonal.
__host__ __device__ inline int needed_rows(int j, int bm, int bn, int tiles_m) {
  const int rows = (j * bn + bn - 1) / bm + 1;
  return rows < tiles_m ? rows : tiles_m;
}

__device__ __forceinline__ Where locate(const Product& p, int tile, int bm, int bn, int per) {
  Where w;
  w.matrix = tile / per;
  int rest = tile - w.matrix * per;
  if (!p.symmetric) {
    w.j = rest / p.tiles_m;
    w.i = rest - w.j * p.tiles_m;
    return w;
  }
  w.j = 0;
  for (int rows = needed_rows(0, bm, bn, p.tiles_m); rest >= rows; rows = needed_rows(++w.j, bm, bn, p.tiles_m)) rest -= rows;
  w.i = rest;
  return w;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// An epilogue box: 32 lines of 64 B. Byte of 16-byte chunk `chunk` (0-3) of a line, swizzled so that threads
// which own a line each, and four threads to a line, both reach 32 banks at once.
__device__ __forceinline__ uint32_t box_at(int line, int chunk) {
  return (uint32_t)(line * 64 + ((chunk ^ ((line >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Transposes the box (the whole warp), 8 x 8 values at a time.
__device__ __forceinline__ void turn_box(uint32_t box, int lane) {
  uint32_t r[4][4];  // [c][q]: the transpose of columns 8 c .. 8 c + 7 of lines 8 q .. 8 q + 7
#pragma unroll
  for (int c = 0; c < 4; ++c)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[c][0]), "=r"(r[c][1]), "=r"(r[c][2]), "=r"(r[c][3])
                 : "r"(box + box_at(lane, c))
                 : "memory");
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(box + box_at(8 * c + (lane & 7), lane >> 3)),
                 "r"(r[c][0]), "r"(r[c][1]), "r"(r[c][2]), "r"(r[c][3])
                 : "memory");
  __syncwarp();
}

__device__ __forceinline__ uint32_t pack_result(int dtype, float x, float y) {
  if (dtype == M3_F16) return pack_half2(x, y);
  const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// A box of 16-bit values to global memory, unit stride along its lines: four threads to a line of 64 B.
// `along`: the lines' elements that exist, from the box on; whole, aligned lines go in words of 16 bytes.
__device__ __forceinline__ void write_box(uint32_t box, int lane, uint16_t* to, int64_t line_stride, int64_t lines, int64_t along) {
  const int at = (lane & 3) * 8;
  uint16_t* first = to + (lane >> 2) * line_stride + at;
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = lds16(box + box_at(8 * i + (lane >> 2), lane & 3));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (8 * i + (lane >> 2) >= lines) break;
    uint16_t* p = first + 8 * i * line_stride;
    if (at + 8 <= along && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      *reinterpret_cast<uint4*>(p) = w[i];
    } else {
      uint64_t low = (uint64_t)w[i].y << 32 | w[i].x, high = (uint64_t)w[i].w << 32 | w[i].z;
#pragma unroll 1
      for (int e = 0; e < 8 && at + e < along; ++e) {
        p[e] = (uint16_t)low;
        low = low >> 16 | high << 48;
        high >>= 16;
      }
    }
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address of `local` in the shared memory of the pair's first CTA.
__device__ __forceinline__ uint32_t in_first(uint32_t local) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(local));
  return r;
}

// The pair's forms of the load (it may complete on the other CTA's barrier), the MMA and the commit (which
// arrives at the same barrier of both CTAs).
__device__ __forceinline__ void pair_load3(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}

// One CTA an SM walks the tiles. kRightByRows: R's tile is given as rows of R ([k][n], the MMA's N-major
// operand); otherwise as rows of R^T ([n][k], K-major), which is how a symmetric product reads its one
// matrix twice. TMA keeps kStages tiles of 64 in k in flight; the accumulators are double-buffered, so
// the epilogue of a tile runs under the next tile's MMAs.
//
// The epilogue's threads own a row of the accumulator each, and its addends and results pass through boxes in
// shared memory, so that four threads share a 64-byte line in global memory: straight from the rows, an
// instruction touches 32 lines, and a 128 x 256 tile took longer to store (7 us) than its MMAs at k = 2560.
// A block is a chain of latencies (about 3000 clocks), so sixteen warps share a tile's: with four, and TMA loads
// and stores of the boxes to wait for, a tile took 8 us.
// 10768 x 2560, five steps: 1242 us, 920 TFLOP/s of the products that symmetry leaves; a step's X X^T takes 78 us, its
// A A 31 and its P X 120 in the loop. P X (430 tiles on 74 pairs, six waves) has 960 K steps of 16 a pair, 128 clocks each
// of the tensor pipe, and takes 186 thousand clocks, at 1.54 GHz: the pipe is busy 64 % of the time. A step takes 133
// clocks once a tile is under way; first loads and the last tile's epilogue take about 16 thousand, and where the rest
// goes has not been found. X X^T and A A have one wave on 55 of the 74 pairs (pipe 52 and 29 % of the time; A A's epilogue
// is as long as its K steps). 128 x 256 tiles of single CTAs took 1490 us against 1298. 4 x 1336 x 256: 128 us,
// fifteen products of about 7 us each, bound by the launches that wait for one another.
template <int BN, bool kRightByRows, bool kPair>
__global__ void __launch_bounds__(Shape<BN, kPair>::kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap left, const __grid_constant__ CUtensorMap right, const Product p) {
  using S = Shape<BN, kPair>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? blockIdx.x & 1 : 0;
  const int first_tile = kPair ? blockIdx.x >> 1 : blockIdx.x, tile_step = kPair ? gridDim.x >> 1 : gridDim.x;
  const uint32_t bars = base + S::kBars;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S::kStages + s); };
  auto acc_full = [&](int b) { return bars + 8u * (2 * S::kStages + b); };
  auto acc_empty = [&](int b) { return bars + 8u * (2 * S::kStages + 2 + b); };
  const uint32_t drained = bars + 8u * (2 * S::kStages + 4);
  const uint32_t slot = bars + 8u * (2 * S::kStages + 5);
  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&left)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&right)) : "memory");
    for (int s = 0; s < S::kStages; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty(s)));
    }
    for (int b = 0; b < 2; ++b) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(acc_full(b)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(acc_empty(b)), "r"((kPair ? 2 : 1) * S::kWarps));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(drained));
    asm volatile("fence.mbarrier_init.release.cluster;");
  }
  if (warp == 1) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(S::kColumns));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(S::kColumns));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // Only now: the block of a kernel after this one, which waits for this one's end, could otherwise come to this SM
    // and take the columns first, and both would wait for good.
    dependents_may_start();
  }
  __syncwarp();
  fence_before();
  if constexpr (kPair) cluster_sync();  // the other CTA's barriers are there
  else __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  const int kblocks = (p.k + kTileK - 1) / kTileK;
  int per = p.tiles_m * p.tiles_n;
  if (p.symmetric) {
    per = 0;
    for (int j = 0; j < p.tiles_n; ++j) per += needed_rows(j, S::kRows, BN, p.tiles_m);
  }
  wait_for_previous();

  if (warp == 0 && lane == 0) {
    int s = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < p.tiles; tile += tile_step) {
      const Where w = locate(p, tile, S::kRows, BN, per);
      const int row = w.i * S::kRows + rank * kTileM, col = w.j * BN + rank * S::kRight;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait(empty(s), phase ^ 1u)) {
          ok = false;
          break;
        }
        const uint32_t at = base + s * (S::kA + S::kB);
        // the pair's loads all complete on the first CTA's barrier, which its MMA thread waits for
        const uint32_t bar = kPair ? in_first(full(s)) : full(s);
        if (rank == 0) mbar_expect_tx(full(s), (kPair ? 2 : 1) * (S::kA + S::kB));
        auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
          if constexpr (kPair) pair_load3(dst, map, x, y, w.matrix, bar);
          else tma_load3(dst, map, x, y, w.matrix, bar);
        };
        load(at, &left, kb * kTileK, row);
        if constexpr (kRightByRows) {
#pragma unroll
          for (int q = 0; q < S::kRight / 64; ++q)
            load(at + S::kA + q * (kTileK * 128), &right, col + 64 * q, kb * kTileK);
        } else {
          load(at + S::kA, &right, kb * kTileK, col);
        }
        ++issued;
        if (++s == S::kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    // Gave up: the copies still in flight land before the block's shared memory goes (the pair's are waited for
    // by its first CTA, and neither leaves before the other).
    if (!ok && rank == 0)
      for (uint32_t q = 0; q < (issued < (uint32_t)S::kStages ? issued : (uint32_t)S::kStages); ++q) {
        if (--s < 0) {
          s = S::kStages - 1;
          phase ^= 1u;
        }
        mbar_wait(full(s), phase);
      }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t id = idesc(S::kRows, BN, false, false, kRightByRows);
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    auto commit = [&](uint32_t bar) {
      if constexpr (kPair) pair_commit(bar);
      else mma_commit(bar);
    };
    for (int tile = first_tile; ok && tile < p.tiles; tile += tile_step) {
      ok = mbar_wait(acc_empty(buf), acc_phase ^ 1u);
      if (!ok) break;
      fence_after();
      const uint32_t acc = tmem + buf * BN;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait(full(s), phase)) {
          ok = false;
          break;
        }
        fence_after();
        const uint32_t at = base + s * (S::kA + S::kB);
        const uint64_t da = sdesc(at, 16, 1024);
        const uint64_t db = kRightByRows ? sdesc(at + S::kA, kTileK * 128, 1024) : sdesc(at + S::kA, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < kTileK / 16; ++kk) {
          const uint64_t ka = sdesc_at(da, kk * 32), kb_ = sdesc_at(db, kk * (kRightByRows ? 2048 : 32));
          if constexpr (kPair) pair_mma(acc, ka, kb_, id, kb > 0 || kk > 0);
          else mma_f16(acc, ka, kb_, id, kb > 0 || kk > 0);
        }
        commit(empty(s));
        if (++s == S::kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      commit(acc_full(buf));
      if (++buf == 2) {
        buf = 0;
        acc_phase ^= 1u;
      }
    }
    if (!ok) {  // the MMAs issued so far end before their memory is given back
      commit(drained);
      mbar_wait(drained, 0);
    }
  } else if (warp >= 2) {
    const int quarter = warp & 3;  // the TMEM lanes that this warp may read
    const int first = (warp - 2) / 4 * S::kBlocks, last = first + S::kBlocks;  // its blocks of 32 columns
    const uint32_t box = base + S::kBoxes + (warp - 2) * kBox;
    int buf = 0;
    uint32_t acc_phase = 0;
    for (int tile = first_tile; tile < p.tiles; tile += tile_step) {
      const Where w = locate(p, tile, S::kRows, BN, per);
      const int row0 = w.i * S::kRows + rank * kTileM + quarter * 32, row = row0 + lane;
      const int64_t matrix = (int64_t)w.matrix * p.m * p.ld;
      // a block that is in the matrix and, of a symmetric product, on the diagonal or above it
      auto needed = [&](int c) {
        const int col = w.j * BN + 32 * c;
        return c < last && row0 < p.m && col < p.n && !(p.symmetric && col < row0);
      };
      int c = first;
      while (c < last && !needed(c)) ++c;
      uint4 hi[4];
      auto fetch = [&](const __half* from, int k) {
        if (from == nullptr || !needed(k)) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int line = 8 * i + (lane >> 2);
          if (row0 + line >= p.m) continue;
          const int64_t at = matrix + (row0 + line) * p.ld + w.j * BN + 32 * k + (lane & 3) * 8;
          hi[i] = *reinterpret_cast<const uint4*>(from + at);
        }
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) hi[i] = make_uint4(0u, 0u, 0u, 0u);
      fetch(p.add, c);
      const float beta =
          p.beta + (p.add_diagonal && row < p.m ? p.add_diagonal[(int64_t)w.matrix * p.m + row] : 0.0f);
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full(buf), acc_phase))) break;
      fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
      for (; needed(c); ++c) {
        const int col = w.j * BN + 32 * c;
        uint32_t r[32];
        M3_TMEM_LD32(acc + 32 * c, r);
        float v[32];
        auto add_term = [&]() {  // through the box: from four threads a line to a thread a line
#pragma unroll
          for (int i = 0; i < 4; ++i) sts16(box + box_at(8 * i + (lane >> 2), lane & 3), hi[i]);
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 word = lds16(box + box_at(lane, q));
            const __half2* h = reinterpret_cast<const __half2*>(&word);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __half22float2(h[e]);
              v[8 * q + 2 * e] = fmaf(beta, f.x, v[8 * q + 2 * e]);
              v[8 * q + 2 * e + 1] = fmaf(beta, f.y, v[8 * q + 2 * e + 1]);
            }
          }
          __syncwarp();
        };
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = p.alpha * __uint_as_float(r[e]);
        if (p.add) add_term();
        if (p.add_lo) {
          fetch(p.add_lo, c);
          add_term();
        }
        fetch(p.add, c + 1);
        const m3_tensor& t = p.result;
        const int64_t there = w.matrix * t.stride[0] + row0 * t.stride[1] + col * t.stride[2];
        const bool by_rows = t.stride[2] == 1, by_cols = t.stride[1] == 1;
        if (p.out == nullptr && (t.dtype == M3_F32 || !(by_rows || by_cols))) {
          // a result that does not go through the box: float32, or unit stride nowhere
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (row < p.m && col + e < p.n) st_t(t, there + lane * t.stride[1] + e * t.stride[2], v[e] * (1.0f / kHold));
          __syncwarp();
          continue;
        }
        if (p.diagonal && col == row0) {
          float d = v[0];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            d = lane == e ? v[e] : d;
            v[e] = lane == e ? 0.0f : v[e];
          }
          if (row < p.m) p.diagonal[(int64_t)w.matrix * p.m + row] = d * (1.0f / kHold);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t word[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = v[8 * q + 2 * e], y = v[8 * q + 2 * e + 1];
            word[e] = p.out ? pack_half2(x, y) : pack_result(t.dtype, x * (1.0f / kHold), y * (1.0f / kHold));
          }
          sts16(box + box_at(lane, q), make_uint4(word[0], word[1], word[2], word[3]));
        }
        __syncwarp();
        const int64_t at = matrix + row0 * p.ld + col;  // the words past n are in the row's padding
        if (p.out) write_box(box, lane, reinterpret_cast<uint16_t*>(p.out + at), p.ld, p.m - row0, 32);
        else if (by_rows) write_box(box, lane, static_cast<uint16_t*>(t.data) + there, t.stride[1], p.m - row0, p.n - col);
        // A symmetric product's block above the diagonal is written mirrored as well (both triangles of one on it are
        // computed), and a transposed result only so.
        if (p.out ? p.symmetric && col > row0 : !by_rows) {
          turn_box(box, lane);
          if (p.out) write_box(box, lane, reinterpret_cast<uint16_t*>(p.out + matrix + col * p.ld + row0), p.ld, p.n - col, 32);
          else write_box(box, lane, static_cast<uint16_t*>(t.data) + there, t.stride[2], p.n - col, p.m - row0);
        }
        if (p.out_lo) {
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t word[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = v[8 * q + 2 * e], y = v[8 * q + 2 * e + 1];
              const uint32_t held = pack_half2(x, y);
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&held));
              word[e] = pack_half2(x - f.x, y - f.y);
            }
            sts16(box + box_at(lane, q), make_uint4(word[0], word[1], word[2], word[3]));
          }
          __syncwarp();
          write_box(box, lane, reinterpret_cast<uint16_t*>(p.out_lo + at), p.ld, p.m - row0, 32);
        }
        __syncwarp();  // the box is free, and the next TMEM read is the whole warp's
      }
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair)
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(acc_empty(buf))) : "memory");
        else
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acc_empty(buf)) : "memory");
      }
      if (++buf == 2) {
        buf = 0;
        acc_phase ^= 1u;
      }
    }
  }
  __syncwarp();
  fence_before();
  if constexpr (kPair) cluster_sync();  // neither CTA leaves while the other's MMAs or arrivals can reach it
  else __syncthreads();
  fence_after();
  if (warp == 1) {
    if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns));
  }
}

// ---- host ----------------------------------------------------------------------------------------

struct Plan {
  int64_t m, n, ldx, lda, bytes, parts, x[2], lo[2], gram, poly, diagonal;
};

Plan plan(const m3_orth_args& a) {
  Plan p;
  p.m = std::min(a.rows, a.cols);
  p.n = std::max(a.rows, a.cols);
  p.ldx = (p.n + 63) / 64 * 64;
  p.lda = (p.m + 63) / 64 * 64;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 1023) / 1024 * 1024;
    return here;
  };
  p.parts = take((int64_t)a.count * kNormParts * 8);
  for (int i = 0; i < 2; ++i) p.x[i] = take((int64_t)a.count * p.m * p.ldx * 2);
  for (int i = 0; i < 2; ++i) p.lo[i] = take((int64_t)a.count * p.m * p.ldx * 2);
  p.gram = take((int64_t)a.count * p.m * p.lda * 2);
  p.poly = take((int64_t)a.count * p.m * p.lda * 2);
  p.diagonal = take((int64_t)a.count * p.m * 4);
  p.bytes = at;
  return p;
}

// A stack of fp16 matrices.
struct Stack {
  __half* data;
  int64_t rows, cols, ld;
};

// Tiles of 64 columns x box_rows rows of a stack; what lies outside reads as 0.
bool encode(CUtensorMap* map, const Stack& t, int count, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)t.cols, (cuuint64_t)t.rows, (cuuint64_t)count};
  const cuuint64_t strides[2] = {(cuuint64_t)t.ld * 2, (cuuint64_t)(t.ld * t.rows) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, t.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t config(dim3 grid, int threads, size_t smem, cudaStream_t stream, cudaLaunchAttribute* chained, bool pair) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  chained->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  chained->val.programmaticStreamSerializationAllowed = 1;
  if (pair) {
    chained[1].id = cudaLaunchAttributeClusterDimension;
    chained[1].val.clusterDim.x = 2;
    chained[1].val.clusterDim.y = chained[1].val.clusterDim.z = 1;
  }
  c.attrs = chained;
  c.numAttrs = pair ? 2 : 1;
  return c;
}

int64_t tile_count(const Product& p, int bm, int bn, int count) {
  const int tm = (p.m + bm - 1) / bm, tn = (p.n + bn - 1) / bn;
  int64_t per = (int64_t)tm * tn;
  if (p.symmetric) {
    per = 0;
    for (int j = 0; j < tn; ++j) per += needed_rows(j, bm, bn, tm);
  }
  return per * count;
}

template <int BN, bool kRightByRows, bool kPair>
cudaError_t launch_product(Product p, const Stack& left, const Stack& right, int count, cudaStream_t stream) {
  using S = Shape<BN, kPair>;
  CUtensorMap ml, mr;
  if (!encode(&ml, left, count, kTileM) || !encode(&mr, right, count, kRightByRows ? kTileK : S::kRight)) return cudaErrorInvalidValue;
  p.tiles_m = (p.m + S::kRows - 1) / S::kRows;
  p.tiles_n = (p.n + BN - 1) / BN;
  p.tiles = (int)tile_count(p, S::kRows, BN, count);
  auto kernel = product_kernel<BN, kRightByRows, kPair>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kBytes);
  if (e != cudaSuccess) return e;
  const int ctas = kPair ? 2 * std::min(p.tiles, sm_count() / 2) : std::min(p.tiles, sm_count());
  cudaLaunchAttribute chained[2];
  const cudaLaunchConfig_t c = config(dim3((unsigned)ctas), S::kThreads, S::kBytes, stream, chained, kPair);
  return cudaLaunchKernelEx(&c, kernel, ml, mr, p);
}

// The widest tile whose tiles still occupy half of the SMs: wide tiles read less from L2 for each product,
// narrow ones keep small stacks off a few SMs. us with the symmetric products / P X in tiles of
//                      64 / 64   64 / 128  64 / 256  128 / 128  128 / 256  256 / 256   the rule's
//   10768 x 2560       2412      1856      1607      1652       1501       1168        256 / 256
//   2048 x 2048        456       372       348       301        275        332         128 / 256
//   8 x 512 x 2048     310       301       296       263        258        303         128 / 256
//   2 x 1024 x 4096    383       325       309       345        328        374         64 / 256
//   1336 x 1336        198       175       199       195        214        261         64 / 128
//   4 x 1336 x 256     124       121       144       140        162        197         64 / 128
//   16 x 256 x 256     99        108       127       122        144        178         64 / 64
//   4 x 1024 x 2048    434       358       338       307        288        344         256 / 256: not the best
//   4 x 700 x 900      180       182       183       200        198        242         128 / 256: not the best
int tile_width(const Product& p, int count) {
  return 4 * tile_count(p, 256, 256, count) >= sm_count() ? 256 : 2 * tile_count(p, 128, 128, count) >= sm_count() ? 128 : 64;
}

template <bool kRightByRows>
cudaError_t launch(const Product& p, const Stack& left, const Stack& right, int count, cudaStream_t stream) {
  switch (tile_width(p, count)) {
    case 256: return launch_product<256, kRightByRows, true>(p, left, right, count, stream);
    case 128: return launch_product<128, kRightByRows, false>(p, left, right, count, stream);
    default: return launch_product<64, kRightByRows, false>(p, left, right, count, stream);
  }
}

cudaError_t run(const m3_orth_args& a, cudaStream_t stream) {
  const Plan pl = plan(a);
  const bool turn = a.rows > a.cols;
  const int m = (int)pl.m, n = (int)pl.n;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace.data);
  auto wide = [&](int64_t at) { return Stack{reinterpret_cast<__half*>(ws + at), m, n, pl.ldx}; };
  const Stack x[2] = {wide(pl.x[0]), wide(pl.x[1])}, lo[2] = {wide(pl.lo[0]), wide(pl.lo[1])};
  const Stack gram = {reinterpret_cast<__half*>(ws + pl.gram), m, m, pl.lda};
  const Stack poly = {reinterpret_cast<__half*>(ws + pl.poly), m, m, pl.lda};
  float* diagonal = reinterpret_cast<float*>(ws + pl.diagonal);
  double* parts = reinterpret_cast<double*>(ws + pl.parts);
  // strides of X's rows and columns in the update
  const int64_t row_stride = a.update.stride[turn ? 2 : 1], col_stride = a.update.stride[turn ? 1 : 2];
  m3_tensor result = a.out;
  if (turn) std::swap(result.stride[1], result.stride[2]);
  // along: the dimension of X whose stride is 1 (columns where neither is); the reads run along it, in runs of 8
  // elements where every run is aligned and whole
  const bool by_rows = col_stride == 1;
  const int64_t along = by_rows ? n : m, across = by_rows ? m : n, across_stride = by_rows ? row_stride : col_stride;
  const int64_t along_stride = by_rows ? col_stride : row_stride;
  const int run_bytes = a.update.dtype == M3_F32 ? 32 : 16;
  const bool vec = along_stride == 1 && along % 8 == 0 && across_stride % 8 == 0 && a.update.stride[0] % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(a.update.data) % run_bytes == 0;
  const bool flat = along_stride == 1 && across_stride == along;  // one run: no division an element
  norm_kernel<<<dim3(kNormParts, a.count), kNormThreads, 0, stream>>>(a, flat ? 1 : across, flat ? across * along : along,
                                                                      across_stride, along_stride, vec, parts);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute chained[2];
  cudaLaunchConfig_t c = config(dim3((unsigned)std::min((pl.n + 63) / 64 * ((pl.m + 63) / 64), (int64_t)std::max(1, 8 * sm_count() / a.count)), a.count), 256,
                                0, stream, chained, false);
  e = cudaLaunchKernelEx(&c, start_kernel, a, (const double*)parts, m, n, pl.ldx, row_stride, col_stride, vec, x[0].data, lo[0].data);
  if (e != cudaSuccess) return e;
  if (a.steps == 0) {
    finish_kernel<<<dim3((unsigned)((pl.m * pl.n + 255) / 256), a.count), 256, 0, stream>>>(
        a, x[0].data, lo[0].data, m, n, pl.ldx, result.stride[1], result.stride[2]);
    return cudaGetLastError();
  }
  for (int t = 0; t < a.steps; ++t) {
    const Stack& now = x[t & 1];
    const bool last = t + 1 == a.steps;
    Product p = {};
    p.m = p.n = m;
    p.k = n;
    p.symmetric = 1;
    p.alpha = 1.0f / kHold;
    p.ld = pl.lda;
    p.out = gram.data;
    e = launch<false>(p, now, now, a.count, stream);
    if (e != cudaSuccess) return e;
    p.k = m;
    p.alpha = a.coefficient[2] / kHold;
    p.beta = a.coefficient[1];
    p.add = gram.data;
    p.diagonal = diagonal;
    p.out = poly.data;
    e = launch<false>(p, gram, gram, a.count, stream);
    if (e != cudaSuccess) return e;
    p = {};
    p.m = p.k = m;
    p.n = n;
    p.alpha = 1.0f / kHold;
    p.beta = a.coefficient[0];
    p.ld = pl.ldx;
    p.add = now.data;
    p.add_lo = t < kLoSteps ? lo[t].data : nullptr;
    p.add_diagonal = diagonal;
    p.out = last ? nullptr : x[(t + 1) & 1].data;
    p.out_lo = !last && t + 1 < kLoSteps ? lo[t + 1].data : nullptr;
    p.result = result;
    e = launch<true>(p, poly, now, a.count, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int check(const m3_orth_args& a) {
  constexpr int64_t kMost = 1 << 20;  // tile coordinates and tile counts stay far inside 32 bits
  if (a.rows <= 0 || a.cols <= 0 || a.rows > kMost || a.cols > kMost || a.count <= 0 || a.count > 65535 ||
      std::min(a.rows, a.cols) > 65536)
    return report_error(M3_ERR_SHAPE, "m3_orthogonalize: 1 to 65535 matrices of at most 65536 x 1048576");
  if (a.steps < 0 || a.steps > 64) return report_error(M3_ERR_ARGUMENT, "m3_orthogonalize: 0 to 64 steps");
  return M3_OK;
}

}  // namespace newton
}  // namespace m3

extern "C" int64_t m3_orthogonalize_workspace_bytes(const m3_orth_args* args) {
  using namespace m3;
  if (args == nullptr) return -report_error(M3_ERR_ARGUMENT, "null argument struct");
  const int rc = newton::check(*args);
  return rc != M3_OK ? -rc : newton::plan(*args).bytes;
}

extern "C" int m3_orthogonalize_tile(const m3_orth_args* args, int product) {
  using namespace m3;
  if (args == nullptr || newton::check(*args) != M3_OK) return 0;
  newton::Product p = {};
  p.m = (int)std::min(args->rows, args->cols);
  p.n = product == 2 ? (int)std::max(args->rows, args->cols) : p.m;
  p.symmetric = product != 2;
  return newton::tile_width(p, args->count);
}

extern "C" int m3_orthogonalize(const m3_orth_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_orth_args& a = *args;
  const int rc = newton::check(a);
  if (rc != M3_OK) return rc;
  if (!a.update.data || !a.out.data || !a.workspace.data)
    return report_error(M3_ERR_ARGUMENT, "m3_orthogonalize: update, out and workspace are required");
  auto fl = [](const m3_tensor& t) { return t.ndim == 3 && t.dtype >= M3_F32 && t.dtype <= M3_BF16; };
  if (!fl(a.update) || !fl(a.out)) return report_error(M3_ERR_DTYPE, "m3_orthogonalize: update and out are 3-D float tensors");
  if (reinterpret_cast<uintptr_t>(a.workspace.data) % 256 != 0)
    return report_error(M3_ERR_LAYOUT, "m3_orthogonalize: the workspace must be 256-byte aligned");
  if (a.device >= 0 && cudaSetDevice(a.device) != cudaSuccess)
    return report_error(M3_ERR_CUDA, "m3_orthogonalize: cannot select the device");
  const cudaError_t e = newton::run(a, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess)
    return report_error(M3_ERR_CUDA, (std::string("m3_orthogonalize launch failed: ") + cudaGetErrorString(e)).c_str());
  return M3_OK;
}
