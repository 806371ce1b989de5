// Newton-Schulz orthogonalisation of optimiser updates, a stack of [rows, cols] matrices.
//
// X_0 = G / |G|_F (0 for G = 0), m <= n after a transposition where rows > cols, then `steps` times
//   A = X X^T,   X <- a X + (b A + c A A) X.
// The squared norm is summed in float64 (a float32 sum of squares overflows above 2e19).
#include <string>

#include "common.cuh"

namespace m3 {

int report_error(int code, const char* msg);

namespace {

constexpr int kNormParts = 64;  // partial sums of squares per matrix

__global__ void __launch_bounds__(256) orth_norm_kernel(const m3_orth_args a, double* parts) {
  __shared__ double warp_part[8];
  const int64_t n = a.rows * a.cols;
  const int64_t base = (int64_t)blockIdx.y * a.update.stride[0];
  double ss = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += 256 * kNormParts) {
    const double v = ld_t(a.update, base + i / a.cols * a.update.stride[1] + i % a.cols * a.update.stride[2]);
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

// x[m][n] = update (or its transpose) / |update|_F
__global__ void __launch_bounds__(256) orth_start_kernel(const m3_orth_args a, const double* parts, float* x) {
  double ss = 0.0;
  for (int p = 0; p < kNormParts; ++p) ss += parts[(int64_t)blockIdx.y * kNormParts + p];
  const double inv = ss > 0.0 ? 1.0 / sqrt(ss) : ss == 0.0 ? 0.0 : ss;
  const bool turn = a.rows > a.cols;
  const int64_t m = turn ? a.cols : a.rows, n = turn ? a.rows : a.cols;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m * n) return;
  const int64_t r = turn ? i % n : i / n, c = turn ? i / n : i % n;
  const double v = ld_t(a.update, (int64_t)blockIdx.y * a.update.stride[0] + r * a.update.stride[1] + c * a.update.stride[2]);
  x[blockIdx.y * m * n + i] = (float)(v * inv);
}

// out = alpha * left * (turn_right ? right^T : right) + beta * add; left [m][k], out / add [m][n]
__global__ void __launch_bounds__(256) orth_product_kernel(const float* left, const float* right, const float* add,
                                                           float* out, int64_t m, int64_t n, int64_t k, bool turn_right,
                                                           float alpha, float beta) {
  __shared__ float ls[16][17], rs[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t row = (int64_t)blockIdx.y * 16 + ty, col = (int64_t)blockIdx.x * 16 + tx;
  left += blockIdx.z * m * k;
  right += blockIdx.z * n * k;
  float acc = 0.0f;
  for (int64_t p = 0; p < k; p += 16) {
    ls[ty][tx] = row < m && p + tx < k ? left[row * k + p + tx] : 0.0f;
    const int64_t other = (int64_t)blockIdx.x * 16 + ty;
    if (turn_right) rs[tx][ty] = other < n && p + tx < k ? right[other * k + p + tx] : 0.0f;
    else rs[ty][tx] = p + ty < k && col < n ? right[(p + ty) * n + col] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 16; ++j) acc = fmaf(ls[ty][j], rs[j][tx], acc);
    __syncthreads();
  }
  if (row < m && col < n) {
    const int64_t i = blockIdx.z * m * n + row * n + col;
    out[i] = alpha * acc + (add ? beta * add[i] : 0.0f);
  }
}

__global__ void __launch_bounds__(256) orth_finish_kernel(const m3_orth_args a, const float* x) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.rows * a.cols) return;
  const int64_t r = i / a.cols, c = i % a.cols;
  const int64_t at = a.rows > a.cols ? c * a.rows + r : i;
  st_t(a.out, (int64_t)blockIdx.y * a.out.stride[0] + r * a.out.stride[1] + c * a.out.stride[2],
       x[blockIdx.y * a.rows * a.cols + at]);
}

struct Plan {
  int64_t m, n, bytes, parts, x0, x1, gram, poly;
};

Plan plan(const m3_orth_args& a) {
  Plan p;
  p.m = a.rows > a.cols ? a.cols : a.rows;
  p.n = a.rows > a.cols ? a.rows : a.cols;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.parts = take((int64_t)a.count * kNormParts * 8);
  p.x0 = take((int64_t)a.count * p.m * p.n * 4);
  p.x1 = take((int64_t)a.count * p.m * p.n * 4);
  p.gram = take((int64_t)a.count * p.m * p.m * 4);
  p.poly = take((int64_t)a.count * p.m * p.m * 4);
  p.bytes = at;
  return p;
}

int check(const m3_orth_args& a) {
  if (a.rows <= 0 || a.cols <= 0 || a.count <= 0 || a.count > 65535)
    return report_error(M3_ERR_SHAPE, "m3_orthogonalize: rows, cols and count (at most 65535) must be positive");
  if (a.steps < 0 || a.steps > 64) return report_error(M3_ERR_ARGUMENT, "m3_orthogonalize: 0 to 64 steps");
  return M3_OK;
}

}  // namespace
}  // namespace m3

extern "C" int64_t m3_orthogonalize_workspace_bytes(const m3_orth_args* args) {
  using namespace m3;
  if (args == nullptr) return -report_error(M3_ERR_ARGUMENT, "null argument struct");
  const int rc = check(*args);
  return rc != M3_OK ? -rc : plan(*args).bytes;
}

extern "C" int m3_orthogonalize(const m3_orth_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_orth_args& a = *args;
  const int rc = check(a);
  if (rc != M3_OK) return rc;
  if (!a.update.data || !a.out.data || !a.workspace.data)
    return report_error(M3_ERR_ARGUMENT, "m3_orthogonalize: update, out and workspace are required");
  auto fl = [](const m3_tensor& t) { return t.ndim == 3 && t.dtype >= M3_F32 && t.dtype <= M3_BF16; };
  if (!fl(a.update) || !fl(a.out)) return report_error(M3_ERR_DTYPE, "m3_orthogonalize: update and out are 3-D float tensors");
  if (a.device >= 0 && cudaSetDevice(a.device) != cudaSuccess)
    return report_error(M3_ERR_CUDA, "m3_orthogonalize: cannot select the device");
  const Plan p = plan(a);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace.data);
  double* parts = reinterpret_cast<double*>(ws + p.parts);
  float *x = reinterpret_cast<float*>(ws + p.x0), *next = reinterpret_cast<float*>(ws + p.x1);
  float *gram = reinterpret_cast<float*>(ws + p.gram), *poly = reinterpret_cast<float*>(ws + p.poly);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 all((unsigned)((a.rows * a.cols + 255) / 256), a.count);
  orth_norm_kernel<<<dim3(kNormParts, a.count), 256, 0, s>>>(a, parts);
  orth_start_kernel<<<all, 256, 0, s>>>(a, parts, x);
  const dim3 square((unsigned)((p.m + 15) / 16), (unsigned)((p.m + 15) / 16), a.count);
  const dim3 wide((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 15) / 16), a.count);
  for (int i = 0; i < a.steps; ++i) {
    orth_product_kernel<<<square, 256, 0, s>>>(x, x, nullptr, gram, p.m, p.m, p.n, true, 1.0f, 0.0f);
    orth_product_kernel<<<square, 256, 0, s>>>(gram, gram, gram, poly, p.m, p.m, p.m, true, a.coefficient[2], a.coefficient[1]);
    orth_product_kernel<<<wide, 256, 0, s>>>(poly, x, x, next, p.m, p.n, p.m, false, 1.0f, a.coefficient[0]);
    float* t = x;
    x = next;
    next = t;
  }
  orth_finish_kernel<<<all, 256, 0, s>>>(a, x);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return report_error(M3_ERR_CUDA, (std::string("m3_orthogonalize launch failed: ") + cudaGetErrorString(e)).c_str());
  return M3_OK;
}
