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

namespace m3 {

int report_error(int code, const char* msg);

namespace {

constexpr int kTile = 64;  // tokens per tile: the training forward keeps the state before each tile

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

template <typename T> __device__ __forceinline__ float ld_elem(const m3_tensor& t, int64_t i) {
  return to_f(static_cast<const T*>(t.data)[i]);
}

// One thread per (batch, channel), one token after another.
template <typename T>
__global__ void __launch_bounds__(64) gated_fwd_kernel(const m3_gated_args a) {
  const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= a.channels) return;
  float h = a.state.data ? static_cast<const float*>(a.state.data)[b * a.state.stride[0] + c * a.state.stride[1]] : 0.0f;
  const uint8_t* rs = a.reset.data ? static_cast<const uint8_t*>(a.reset.data) + b * a.reset.stride[0] : nullptr;
  for (int64_t t = 0; t < a.length; ++t) {
    if (a.carry.data && t % kTile == 0)
      static_cast<float*>(a.carry.data)[b * a.carry.stride[0] + t / kTile * a.carry.stride[1] + c] = h;
    float keep, lose;
    keep_lose(ld_elem<T>(a.forget, b * a.forget.stride[0] + t * a.forget.stride[1] + c * a.forget.stride[2]), keep, lose);
    if (rs && rs[t * a.reset.stride[1]]) h = 0.0f;
    h = keep * h + lose * ld_elem<T>(a.value, b * a.value.stride[0] + t * a.value.stride[1] + c * a.value.stride[2]);
    float y = h;
    if (a.gate.data) {
      const float g = ld_elem<T>(a.gate, b * a.gate.stride[0] + t * a.gate.stride[1] + c * a.gate.stride[2]);
      y *= g * sigmoid_approx(g);
    }
    static_cast<T*>(a.y.data)[b * a.y.stride[0] + t * a.y.stride[1] + c * a.y.stride[2]] = from_f<T>(y);
  }
  static_cast<float*>(a.out_state.data)[b * a.out_state.stride[0] + c * a.out_state.stride[1]] = h;
}

// The same from the back, tile by tile: the tile's states are recomputed from the state before it.
template <typename T>
__global__ void __launch_bounds__(64) gated_bwd_kernel(const m3_gated_args a) {
  const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= a.channels) return;
  const uint8_t* rs = a.reset.data ? static_cast<const uint8_t*>(a.reset.data) + b * a.reset.stride[0] : nullptr;
  float in = a.dstate.data ? static_cast<const float*>(a.dstate.data)[b * a.dstate.stride[0] + c * a.dstate.stride[1]] : 0.0f;
  float before[kTile];
  for (int64_t t0 = (a.length - 1) / kTile * kTile; t0 >= 0; t0 -= kTile) {
    const int n = (int)(a.length - t0 < kTile ? a.length - t0 : kTile);
    float h = static_cast<const float*>(a.carry.data)[b * a.carry.stride[0] + t0 / kTile * a.carry.stride[1] + c];
    for (int i = 0; i < n; ++i) {
      const int64_t t = t0 + i;
      if (rs && rs[t * a.reset.stride[1]]) h = 0.0f;
      before[i] = h;
      float keep, lose;
      keep_lose(ld_elem<T>(a.forget, b * a.forget.stride[0] + t * a.forget.stride[1] + c * a.forget.stride[2]), keep, lose);
      h = keep * h + lose * ld_elem<T>(a.value, b * a.value.stride[0] + t * a.value.stride[1] + c * a.value.stride[2]);
    }
    for (int i = n - 1; i >= 0; --i) {
      const int64_t t = t0 + i;
      const float v = ld_elem<T>(a.value, b * a.value.stride[0] + t * a.value.stride[1] + c * a.value.stride[2]);
      float keep, lose;
      keep_lose(ld_elem<T>(a.forget, b * a.forget.stride[0] + t * a.forget.stride[1] + c * a.forget.stride[2]), keep, lose);
      float dh = ld_elem<T>(a.dy, b * a.dy.stride[0] + t * a.dy.stride[1] + c * a.dy.stride[2]);
      if (a.gate.data) {
        const float g = ld_elem<T>(a.gate, b * a.gate.stride[0] + t * a.gate.stride[1] + c * a.gate.stride[2]);
        const float s = sigmoid_approx(g);
        const float ht = keep * before[i] + lose * v;
        static_cast<T*>(a.dgate.data)[b * a.dgate.stride[0] + t * a.dgate.stride[1] + c * a.dgate.stride[2]] =
            from_f<T>(dh * ht * (s * (1.0f + g * (1.0f - s))));
        dh *= g * s;
      }
      const float G = dh + in;
      static_cast<T*>(a.dvalue.data)[b * a.dvalue.stride[0] + t * a.dvalue.stride[1] + c * a.dvalue.stride[2]] =
          from_f<T>(G * lose);
      static_cast<T*>(a.dforget.data)[b * a.dforget.stride[0] + t * a.dforget.stride[1] + c * a.dforget.stride[2]] =
          from_f<T>(G * (before[i] - v) * (keep * lose));
      in = rs && rs[t * a.reset.stride[1]] ? 0.0f : keep * G;
    }
  }
  if (a.dinitial.data) static_cast<float*>(a.dinitial.data)[b * a.dinitial.stride[0] + c * a.dinitial.stride[1]] = in;
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

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
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
  const dim3 grid((a.channels + 63) / 64, a.batch);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a.value.dtype) {
    case M3_BF16: gated_fwd_kernel<__nv_bfloat16><<<grid, 64, 0, s>>>(a); break;
    case M3_F16: gated_fwd_kernel<__half><<<grid, 64, 0, s>>>(a); break;
    default: gated_fwd_kernel<float><<<grid, 64, 0, s>>>(a); break;
  }
  return launched("gated scan");
}

extern "C" int m3_gated_scan_bwd(const m3_gated_args* args, void* stream) {
  using namespace m3;
  if (args == nullptr) return report_error(M3_ERR_ARGUMENT, "null argument struct");
  const m3_gated_args& a = *args;
  const int rc = check(a, true);
  if (rc != M3_OK) return rc;
  const dim3 grid((a.channels + 63) / 64, a.batch);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a.value.dtype) {
    case M3_BF16: gated_bwd_kernel<__nv_bfloat16><<<grid, 64, 0, s>>>(a); break;
    case M3_F16: gated_bwd_kernel<__half><<<grid, 64, 0, s>>>(a); break;
    default: gated_bwd_kernel<float><<<grid, 64, 0, s>>>(a); break;
  }
  return launched("gated scan backward");
}
