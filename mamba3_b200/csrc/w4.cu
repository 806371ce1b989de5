// Few-row projection with 4-bit weights: y[r][o] = sum_i x[r][i] s[o][g] (q[o][i] - z[o][g]), g = i / group.
//
// Codes are packed two to a byte, the even column in the low half, rows of (in_dim + 1) / 2 bytes;
// scales (and zero points, 8 where there are none) are one value per row and group. q - 8 is exact
// in 16 bits, sums are float32, y is rounded once.
#include <string>

#include "common.cuh"

namespace m3 {

int report_error(int code, const char* msg);

namespace {

constexpr int kW4Threads = 256;

// One warp per output: any sizes, strides and alignments.
template <typename T>
__global__ void __launch_bounds__(kW4Threads) w4_kernel(const m3_w4_args a) {
  const int lane = threadIdx.x & 31;
  const int64_t o = (int64_t)blockIdx.x * (kW4Threads / 32) + (threadIdx.x >> 5);
  const int64_t r = blockIdx.y;
  if (o >= a.out_dim) return;
  const uint8_t* q = static_cast<const uint8_t*>(a.codes.data) + o * a.codes.stride[0];
  const T* x = static_cast<const T*>(a.x.data) + r * a.x.stride[0];
  float acc = 0.0f;
  for (int64_t i = lane; i < a.in_dim; i += 32) {
    const int64_t g = i / a.group;
    const float s = ld_t(a.scales, o * a.scales.stride[0] + g * a.scales.stride[1]);
    const float z = a.zeros.data ? ld_t(a.zeros, o * a.zeros.stride[0] + g * a.zeros.stride[1]) : 8.0f;
    const int byte = q[(i >> 1) * a.codes.stride[1]];
    const float w = (float)((i & 1) ? byte >> 4 : byte & 15) - z;
    acc = fmaf(to_f(x[i * a.x.stride[1]]), w * s, acc);
  }
  acc = warp_sum(acc);
  if (lane == 0) static_cast<T*>(a.y.data)[r * a.y.stride[0] + o * a.y.stride[1]] = from_f<T>(acc);
}

}  // namespace
}  // namespace m3

extern "C" int m3_linear_w4(const m3_w4_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_w4_args& a = *args;
  if (a.rows <= 0 || a.out_dim <= 0 || a.in_dim <= 0)
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: rows, out_dim and in_dim must be positive");
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
  if (a.rows > 65535) return report_error(M3_ERR_SHAPE, "m3_linear_w4: rows above 65535");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((a.out_dim + 7) / 8), (unsigned)a.rows);
  if (a.x.dtype == M3_BF16) w4_kernel<__nv_bfloat16><<<grid, kW4Threads, 0, s>>>(a);
  else w4_kernel<__half><<<grid, kW4Threads, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return report_error(M3_ERR_CUDA, (std::string("m3_linear_w4 launch failed: ") + cudaGetErrorString(e)).c_str());
  return M3_OK;
}
