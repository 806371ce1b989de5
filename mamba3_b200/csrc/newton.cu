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
int read_newton_error(int clear) {
  int host = 0;
  if (cudaMemcpyFromSymbol(&host, g_device_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return host;
}

namespace newton {

using namespace umma;

constexpr float kHold = 256.0f;   // stored entries are the matrix's times this
constexpr int kNormParts = 256;   // partial sums of squares per matrix
constexpr int kLoSteps = 2;       // X_0 .. X_{kLoSteps - 1} keep their rounding residue

__device__ __forceinline__ void dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- the norm and X_0 ----------------------------------------------------------------------------

// Sums of squares over rows r = part, part + kNormParts, ... of one matrix.
__global__ void __launch_bounds__(256) norm_kernel(const m3_orth_args a, int64_t rows, int64_t cols, int64_t row_stride,
                                                   int64_t col_stride, double* parts) {
  __shared__ double warp_part[8];
  dependents_may_start();
  const int64_t base = (int64_t)blockIdx.y * a.update.stride[0];
  double ss = 0.0;
  for (int64_t r = blockIdx.x; r < rows; r += kNormParts)
    for (int64_t c = threadIdx.x; c < cols; c += 256) {
      const double v = ld_t(a.update, base + r * row_stride + c * col_stride);
      ss += v * v;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += warp_part[w];
    parts[(int64_t)blockIdx.y * kNormParts + blockIdx.x] = t;
  }
}

// hi + lo = 256 G / |G| as [m][ld], 64 x 64 elements a block, through shared memory: the reads run along
// the dimension of G whose stride is 1, the writes along X's rows.
__global__ void __launch_bounds__(256) start_kernel(const m3_orth_args a, const double* parts, int m, int n, int64_t ld,
                                                    int64_t row_stride, int64_t col_stride, __half* hi, __half* lo) {
  __shared__ float tile[64][65];
  __shared__ float factor[2];
  const int tid = threadIdx.x;
  dependents_may_start();
  wait_for_previous();
  if (tid < 32) {
    double ss = 0.0;
    for (int p = tid; p < kNormParts; p += 32) ss += parts[(int64_t)blockIdx.z * kNormParts + p];
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
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const int64_t base = (int64_t)blockIdx.z * a.update.stride[0];
  const bool along_rows = col_stride != 1;  // G's unit stride runs down X's columns
  for (int i = tid; i < 64 * 64; i += 256) {
    const int r = along_rows ? i & 63 : i >> 6, c = along_rows ? i >> 6 : i & 63;
    tile[r][c] = r0 + r < m && c0 + c < n ? ld_t(a.update, base + (r0 + r) * row_stride + (c0 + c) * col_stride) : 0.0f;
  }
  __syncthreads();
  const float f0 = factor[0], f1 = factor[1];
  for (int i = tid; i < 64 * 8; i += 256) {
    const int r = i >> 3, c = (i & 7) * 8;
    if (r0 + r >= m) continue;
    alignas(16) __half h[8], l[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = tile[r][c + e] * f0 * f1;
      h[e] = __float2half_rn(v);
      l[e] = __float2half_rn(v - __half2float(h[e]));
    }
    // ld is a multiple of 64: the columns past n are there
    const int64_t at = ((int64_t)blockIdx.z * m + r0 + r) * ld + c0 + c;
    *reinterpret_cast<uint4*>(hi + at) = *reinterpret_cast<const uint4*>(h);
    *reinterpret_cast<uint4*>(lo + at) = *reinterpret_cast<const uint4*>(l);
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
  int64_t ld;                            // row stride of add, out and their residues; matrices m * ld apart
  const __half *add, *add_lo;            // null: no such term
  const float* add_diagonal;             // [matrix][m], joins beta row by row; null: none
  float* diagonal;                       // [matrix][m]: the diagonal goes there and out has 0 instead; null: it stays
  __half *out, *out_lo;                  // out null: the result goes to `result`
  m3_tensor result;                      // strides (matrix, row, column) of X's orientation, values / 256
};

constexpr int kTileM = 128, kTileK = 64;
constexpr int kProductThreads = 192;  // warp 0 loads, warp 1 issues the MMAs, warps 2-5 run the epilogue

template <int BN> struct Shape {
  static constexpr uint32_t kA = kTileM * kTileK * 2, kB = BN * kTileK * 2;
  static constexpr int kStages = 196608 / (kA + kB);  // 4, 6 or 8 stages of 48, 32 or 24 KB
  static constexpr uint32_t kBars = kStages * (kA + kB);
  static constexpr uint32_t kBytes = kBars + 256 + 1024;  // + alignment slack
  static constexpr uint32_t kColumns = 2 * BN;            // two accumulators
};

struct Where {
  int matrix, i, j;  // which matrix of the stack, tile row, tile column
};

// Tile rows (of 128) of tile column j that a symmetric product needs: those with an element on or
// above the diagonal.
__host__ __device__ inline int needed_rows(int j, int bn, int tiles_m) {
  const int rows = (j * bn + bn - 1) / kTileM + 1;
  return rows < tiles_m ? rows : tiles_m;
}

__device__ __forceinline__ Where locate(const Product& p, int tile, int bn, int per) {
  Where w;
  w.matrix = tile / per;
  int rest = tile - w.matrix * per;
  if (!p.symmetric) {
    w.j = rest / p.tiles_m;
    w.i = rest - w.j * p.tiles_m;
    return w;
  }
  w.j = 0;
  for (int rows = needed_rows(0, bn, p.tiles_m); rest >= rows; rows = needed_rows(++w.j, bn, p.tiles_m)) rest -= rows;
  w.i = rest;
  return w;
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 values of row `row`, columns col .. col + 31, to the caller's tensor.
__device__ __forceinline__ void store_result(const m3_tensor& t, int64_t base, int row, int col, int n, const float* v) {
  const int64_t at = base + row * t.stride[1] + col * t.stride[2];
  if (t.stride[2] == 1 && col + 32 <= n && t.dtype != M3_F32 && ((reinterpret_cast<uintptr_t>(t.data) + 2 * at) & 15) == 0) {
    uint4* to = reinterpret_cast<uint4*>(static_cast<__half*>(t.data) + at);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = v[8 * q + 2 * e], y = v[8 * q + 2 * e + 1];
        if (t.dtype == M3_F16) {
          w[e] = pack_half2(x, y);
        } else {
          const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
          w[e] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      to[q] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (col + e < n) st_t(t, at + e * t.stride[2], v[e]);
}

// One CTA an SM walks the tiles of 128 x BN. kRightByRows: R's tile is given as rows of R ([k][n], the
// MMA's N-major operand); otherwise as rows of R^T ([n][k], K-major), which is how a symmetric product
// reads its one matrix twice. TMA keeps kStages tiles of 64 in k in flight; the accumulators are
// double-buffered, so the epilogue of a tile runs under the next tile's MMAs.
template <int BN, bool kRightByRows>
__global__ void __launch_bounds__(kProductThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap left, const __grid_constant__ CUtensorMap right, const Product p) {
  using S = Shape<BN>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bars = base + S::kBars;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (S::kStages + s); };
  auto acc_full = [&](int b) { return bars + 8u * (2 * S::kStages + b); };
  auto acc_empty = [&](int b) { return bars + 8u * (2 * S::kStages + 2 + b); };
  const uint32_t drained = bars + 8u * (2 * S::kStages + 4);
  const uint32_t slot = bars + 8u * (2 * S::kStages + 5);
  dependents_may_start();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(S::kColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty(s)));
    }
    for (int b = 0; b < 2; ++b) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(acc_full(b)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" ::"r"(acc_empty(b)));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(drained));
    asm volatile("fence.mbarrier_init.release.cluster;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  const int kblocks = (p.k + kTileK - 1) / kTileK;
  int per = p.tiles_m * p.tiles_n;
  if (p.symmetric) {
    per = 0;
    for (int j = 0; j < p.tiles_n; ++j) per += needed_rows(j, BN, p.tiles_m);
  }
  wait_for_previous();

  if (warp == 0 && lane == 0) {
    int s = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
      const Where w = locate(p, tile, BN, per);
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait(empty(s), phase ^ 1u)) {
          ok = false;
          break;
        }
        const uint32_t at = base + s * (S::kA + S::kB);
        mbar_expect_tx(full(s), S::kA + S::kB);
        tma_load3(at, &left, kb * kTileK, w.i * kTileM, w.matrix, full(s));
        if constexpr (kRightByRows) {
#pragma unroll
          for (int q = 0; q < BN / 64; ++q)
            tma_load3(at + S::kA + q * (kTileK * 128), &right, w.j * BN + 64 * q, kb * kTileK, w.matrix, full(s));
        } else {
          tma_load3(at + S::kA, &right, kb * kTileK, w.j * BN, w.matrix, full(s));
        }
        ++issued;
        if (++s == S::kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok)  // gave up: the copies still in flight land before the block's shared memory goes
      for (uint32_t q = 0; q < (issued < (uint32_t)S::kStages ? issued : (uint32_t)S::kStages); ++q) {
        if (--s < 0) {
          s = S::kStages - 1;
          phase ^= 1u;
        }
        mbar_wait(full(s), phase);
      }
  } else if (warp == 1 && lane == 0) {
    const uint32_t id = idesc(kTileM, BN, false, false, kRightByRows);
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < p.tiles; tile += gridDim.x) {
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
        for (int kk = 0; kk < kTileK / 16; ++kk)
          mma_f16(acc, sdesc_at(da, kk * 32), sdesc_at(db, kk * (kRightByRows ? 2048 : 32)), id, kb > 0 || kk > 0);
        mma_commit(empty(s));
        if (++s == S::kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      mma_commit(acc_full(buf));
      if (++buf == 2) {
        buf = 0;
        acc_phase ^= 1u;
      }
    }
    if (!ok) {  // the MMAs issued so far end before their memory is given back
      mma_commit(drained);
      mbar_wait(drained, 0);
    }
  } else if (warp >= 2) {
    const int quarter = warp & 3;  // the TMEM lanes that this warp may read
    int buf = 0;
    uint32_t acc_phase = 0;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const Where w = locate(p, tile, BN, per);
      const int row = w.i * kTileM + quarter * 32 + lane;
      const int64_t at = (int64_t)w.matrix * p.m * p.ld;
      const int64_t row_of_stack = (int64_t)w.matrix * p.m + row;
      const float beta = p.beta + (p.add_diagonal && row < p.m ? p.add_diagonal[row_of_stack] : 0.0f);
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full(buf), acc_phase))) break;
      fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
      for (int c = 0; c < BN / 32; ++c) {
        const int col = w.j * BN + 32 * c;
        __syncwarp();  // the TMEM read below is the whole warp's
        // (the whole warp agrees) nothing of these columns is in the matrix, or on or above the diagonal
        if (col >= p.n || (p.symmetric && col + 31 < row - lane)) continue;
        uint32_t r[32];
        M3_TMEM_LD32(acc + 32 * c, r);
        tmem_wait_ld();
        if (row >= p.m) continue;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = p.alpha * __uint_as_float(r[e]);
        const int64_t here = at + row * p.ld + col;  // ld is a multiple of 64 and col of 32: 16-byte aligned,
                                                     // and the columns past n are there
        auto add_term = [&](const __half* from) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 word = *reinterpret_cast<const uint4*>(from + here + 8 * q);
            const __half2* h = reinterpret_cast<const __half2*>(&word);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __half22float2(h[e]);
              v[8 * q + 2 * e] = fmaf(beta, f.x, v[8 * q + 2 * e]);
              v[8 * q + 2 * e + 1] = fmaf(beta, f.y, v[8 * q + 2 * e + 1]);
            }
          }
        };
        if (p.add) add_term(p.add);
        if (p.add_lo) add_term(p.add_lo);
        if (p.out == nullptr) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] *= 1.0f / kHold;
          store_result(p.result, w.matrix * p.result.stride[0], row, col, p.n, v);
          continue;
        }
        if (p.diagonal && row >= col && row < col + 32) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (col + e == row) {
              p.diagonal[row_of_stack] = v[e] * (1.0f / kHold);
              v[e] = 0.0f;
            }
        }
        if (!p.symmetric || col >= row) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t word[4], rest[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = v[8 * q + 2 * e], y = v[8 * q + 2 * e + 1];
              word[e] = pack_half2(x, y);
              const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&word[e]));
              rest[e] = pack_half2(x - held.x, y - held.y);
            }
            *reinterpret_cast<uint4*>(p.out + here + 8 * q) = make_uint4(word[0], word[1], word[2], word[3]);
            if (p.out_lo)
              *reinterpret_cast<uint4*>(p.out_lo + here + 8 * q) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (col + e >= row) p.out[here + e] = __float2half_rn(v[e]);
        }
        if (p.symmetric) {  // the mirrored elements: 32 neighbouring rows are 32 neighbouring columns there
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (col + e > row && col + e < p.n) p.out[at + (col + e) * p.ld + row] = __float2half_rn(v[e]);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acc_empty(buf)) : "memory");
      if (++buf == 2) {
        buf = 0;
        acc_phase ^= 1u;
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns));
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

// A stack of [rows][cols] fp16 matrices (row stride ld), tiles of 64 columns x box_rows rows; what lies
// outside reads as 0.
bool encode(CUtensorMap* map, const __half* data, int64_t rows, int64_t cols, int64_t ld, int count, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)count};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(data), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t config(dim3 grid, int threads, size_t smem, cudaStream_t stream, cudaLaunchAttribute* chained) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  chained->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  chained->val.programmaticStreamSerializationAllowed = 1;
  c.attrs = chained;
  c.numAttrs = 1;
  return c;
}

int64_t tile_count(const Product& p, int bn, int count) {
  const int tm = (p.m + kTileM - 1) / kTileM, tn = (p.n + bn - 1) / bn;
  int64_t per = (int64_t)tm * tn;
  if (p.symmetric) {
    per = 0;
    for (int j = 0; j < tn; ++j) per += needed_rows(j, bn, tm);
  }
  return per * count;
}

template <int BN, bool kRightByRows>
cudaError_t launch_product(Product p, const __half* left, int64_t left_ld, const __half* right, int64_t right_ld, int count,
                           cudaStream_t stream) {
  CUtensorMap ml, mr;
  if (!encode(&ml, left, p.m, p.k, left_ld, count, kTileM)) return cudaErrorInvalidValue;
  if (!(kRightByRows ? encode(&mr, right, p.k, p.n, right_ld, count, kTileK) : encode(&mr, right, p.n, p.k, right_ld, count, BN)))
    return cudaErrorInvalidValue;
  p.tiles_m = (p.m + kTileM - 1) / kTileM;
  p.tiles_n = (p.n + BN - 1) / BN;
  p.tiles = (int)tile_count(p, BN, count);
  auto kernel = product_kernel<BN, kRightByRows>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<BN>::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute chained;
  const cudaLaunchConfig_t c = config(dim3((unsigned)std::min(p.tiles, sm_count())), kProductThreads, Shape<BN>::kBytes, stream, &chained);
  return cudaLaunchKernelEx(&c, kernel, ml, mr, p);
}

// The widest tile whose tiles still occupy half of the SMs: a 128 x 256 tile reads 96 B of shared memory
// a clock at the full MMA rate and a 128 x 128 one 128 B (the port's limit), but narrow tiles keep
// small stacks off a few SMs.
template <bool kRightByRows>
cudaError_t launch(const Product& p, const __half* left, int64_t left_ld, const __half* right, int64_t right_ld, int count,
                   cudaStream_t stream) {
  if (2 * tile_count(p, 256, count) >= sm_count())
    return launch_product<256, kRightByRows>(p, left, left_ld, right, right_ld, count, stream);
  if (2 * tile_count(p, 128, count) >= sm_count())
    return launch_product<128, kRightByRows>(p, left, left_ld, right, right_ld, count, stream);
  return launch_product<64, kRightByRows>(p, left, left_ld, right, right_ld, count, stream);
}

cudaError_t run(const m3_orth_args& a, cudaStream_t stream) {
  const Plan pl = plan(a);
  const bool turn = a.rows > a.cols;
  const int m = (int)pl.m, n = (int)pl.n;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace.data);
  auto half_at = [&](int64_t at) { return reinterpret_cast<__half*>(ws + at); };
  double* parts = reinterpret_cast<double*>(ws + pl.parts);
  // strides of X's rows and columns in the update
  const int64_t row_stride = a.update.stride[turn ? 2 : 1], col_stride = a.update.stride[turn ? 1 : 2];
  m3_tensor result = a.out;
  if (turn) std::swap(result.stride[1], result.stride[2]);
  // the norm's rows run over the dimension whose stride is not 1
  const bool by_rows = col_stride == 1;
  norm_kernel<<<dim3(kNormParts, a.count), 256, 0, stream>>>(a, by_rows ? m : n, by_rows ? n : m, by_rows ? row_stride : col_stride,
                                                             by_rows ? col_stride : row_stride, parts);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute chained;
  cudaLaunchConfig_t c = config(dim3((n + 63) / 64, (m + 63) / 64, a.count), 256, 0, stream, &chained);
  e = cudaLaunchKernelEx(&c, start_kernel, a, (const double*)parts, m, n, pl.ldx, row_stride, col_stride, half_at(pl.x[0]),
                         half_at(pl.lo[0]));
  if (e != cudaSuccess) return e;
  if (a.steps == 0) {
    finish_kernel<<<dim3((unsigned)((pl.m * pl.n + 255) / 256), a.count), 256, 0, stream>>>(
        a, half_at(pl.x[0]), half_at(pl.lo[0]), m, n, pl.ldx, result.stride[1], result.stride[2]);
    return cudaGetLastError();
  }
  for (int t = 0; t < a.steps; ++t) {
    const __half* x = half_at(pl.x[t & 1]);
    Product gram = {};
    gram.m = gram.n = m;
    gram.k = n;
    gram.symmetric = 1;
    gram.alpha = 1.0f / kHold;
    gram.ld = pl.lda;
    gram.out = half_at(pl.gram);
    e = launch<false>(gram, x, pl.ldx, x, pl.ldx, a.count, stream);
    if (e != cudaSuccess) return e;
    Product poly = gram;
    poly.k = m;
    poly.alpha = a.coefficient[2] / kHold;
    poly.beta = a.coefficient[1];
    poly.add = half_at(pl.gram);
    poly.out = half_at(pl.poly);
    poly.diagonal = reinterpret_cast<float*>(ws + pl.diagonal);
    e = launch<false>(poly, half_at(pl.gram), pl.lda, half_at(pl.gram), pl.lda, a.count, stream);
    if (e != cudaSuccess) return e;
    Product next = {};
    next.m = next.k = m;
    next.n = n;
    next.alpha = 1.0f / kHold;
    next.beta = a.coefficient[0];
    next.ld = pl.ldx;
    next.add = x;
    next.add_diagonal = poly.diagonal;
    next.add_lo = t < kLoSteps ? half_at(pl.lo[t]) : nullptr;
    if (t + 1 < a.steps) {
      next.out = half_at(pl.x[(t + 1) & 1]);
      next.out_lo = t + 1 < kLoSteps ? half_at(pl.lo[t + 1]) : nullptr;
    } else {
      next.result = result;
    }
    e = launch<true>(next, half_at(pl.poly), pl.lda, x, pl.ldx, a.count, stream);
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
