// Few-row projection with 4-bit weights: y[r][o] = sum_i x[r][i] s[o][g] (q[o][i] - z[o][g]), g = i / group.
//
// Codes are packed two to a byte, the even column in the low half, rows of (in_dim + 1) / 2 bytes;
// scales (and zero points, 8 where there are none) are one value per row and group.
//
// What bounds it is the stream of the codes, O I / 2 bytes, and their conversion on the way: at the copy rate an SM has
// about 2.7 instructions of a lane for a code, a conversion to float32 and a multiply-add take as many. So the
// products go to the warp-level tensor instruction (m16n8k16: 16 outputs x 8 rows of x), whose 16-bit operands take
// two codes at a time: bits of (1024 + code) less 1032 is code - 8 exactly (in bf16: 128 and 136; the use of an exponent's
// free bits for this is Kim, Henry, Fahim and Awadalla's, 2022). Which column goes
// where in a product is free as long as both operands agree, so the codes are used as they lie in memory: four
// threads share an output row, and of every group a thread has group / 4 neighbouring columns, one load of 4, 8 or
// 16 bytes. Products of 16-bit values by code - 8 are exact, sums float32, scaled group by group:
//   y = sum_g s (sum x (q - 8) - (z - 8) sum x),
// the sums of x by products with ones; y is rounded once. That form loses two things: with an infinity in x it is inf - inf
// where a code and its zero point are on one side of 8, and sum x (q - 8) can pass float32's range where s would bring it
// back. Both leave a sum that is not finite, and such an output is taken again term by term, s (q - z) first.
#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "umma.cuh"

namespace m3 {

int report_error(int code, const char* msg);

// The error word of this unit's bounded waits, for m3_device_error(); the device is synchronised.
int read_w4_error(int clear) { return read_unit_error(clear); }

namespace {

constexpr int kSlab = 128;  // columns that a warp takes at a time, 4 words of 8 codes a thread and output row

// ---- codes ---------------------------------------------------------------------------------------

// (v & mask) | bits, in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
  return r;
}

// Two codes to two values code - 8 in T: bytes 0 and 2 of v hold them in their low halves.
template <typename T> __device__ __forceinline__ uint32_t open2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t w = and_or(v, 0x000F000Fu, 0x64006400u);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6408)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t w = and_or(v, 0x000F000Fu, 0x43004300u);
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

// kCount words of a row of `bytes` bytes from byte `at` on, any alignment; bytes past the row are 0. Where they lie
// inside the row, with what an aligned word more has, they come as aligned words, shifted into place.
template <int kCount>
__device__ __forceinline__ void row_words(const uint8_t* row, int64_t step, int64_t at, int64_t bytes, uint32_t* to) {
  const uint8_t* from = row + at;
  const int off = (int)(reinterpret_cast<uintptr_t>(from) & 3);
  if (step == 1 && at >= off && at + 4 * kCount + (off ? 4 - off : 0) <= bytes) {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(from - off);
    uint32_t held[kCount + 1];
#pragma unroll
    for (int i = 0; i < kCount; ++i) held[i] = words[i];
    held[kCount] = off ? words[kCount] : 0u;
#pragma unroll
    for (int i = 0; i < kCount; ++i) to[i] = __funnelshift_r(held[i], held[i + 1], 8 * off);
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      uint32_t v = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (at + 4 * i + b < bytes) v |= (uint32_t)row[(at + 4 * i + b) * step] << (8 * b);
      to[i] = v;
    }
  }
}

// A value of a type known at run time, by its bits. What is fetched ahead stays bits until it is used: a conversion would
// wait for the load.
__device__ __forceinline__ float widen(uint32_t v, int type) {
  return type == M3_F32 ? __uint_as_float(v) : type == M3_BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half((uint16_t)v));
}
__device__ __forceinline__ uint32_t bits(const uint8_t* at, int type) {
  return type == M3_F32 ? *reinterpret_cast<const uint32_t*>(at) : *reinterpret_cast<const uint16_t*>(at);
}

// Four bytes of a row from byte `at` on, which may lie before it or past it: 0 there.
__device__ __noinline__ uint32_t edge_word(const uint8_t* row, int64_t step, int64_t at, int64_t bytes) {
  uint32_t v = 0;
  for (int b = 0; b < 4; ++b)
    if (at + b >= 0 && at + b < bytes) v |= (uint32_t)row[(at + b) * step] << (8 * b);
  return v;
}

// A warp's 16 output rows, as a thread sees them: rows g and g + 8 (past the end, the last one again: not written).
// kFast: codes in whole aligned words, scales and zeros in 16 bits with unit stride along a row, whole groups: read
// group by group. Otherwise as aligned words around a row's own start, shifted into place where they are used, and byte
// by byte at the tensor's ends or where a row's bytes lie apart.
template <typename T, int kWords, bool kFast, bool kZeros> struct Weight {
  static constexpr int kGroup = 32 * kWords, kPerSlab = kSlab / kGroup, kHeld = kWords + (kFast ? 0 : 1);
  struct Slab {
    uint32_t code[2][kPerSlab][kHeld];
    uint32_t scale[2][kPerSlab], zero[2][kZeros ? kPerSlab : 1];  // bits
  };
  const m3_w4_args& a;
  const uint8_t *code[2], *scale[2], *zero[2];
  int t, in_dim, slabs, type, size;
  int off[2];

  __device__ __forceinline__ Weight(const m3_w4_args& args, int64_t o0, int lane) : a(args), t(lane & 3), in_dim((int)args.in_dim) {
    slabs = (in_dim + kSlab - 1) / kSlab;
    type = a.scales.dtype;
    size = !kFast && type == M3_F32 ? 4 : 2;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = min(o0 + (lane >> 2) + 8 * r, a.out_dim - 1);
      code[r] = static_cast<const uint8_t*>(a.codes.data) + row * a.codes.stride[0] + (kFast ? 4 * kWords * t : 0);
      off[r] = !kFast && a.codes.stride[1] == 1 ? (int)(reinterpret_cast<uintptr_t>(code[r]) & 3) : 0;
      scale[r] = static_cast<const uint8_t*>(a.scales.data) + row * a.scales.stride[0] * size;
      if (kZeros) zero[r] = static_cast<const uint8_t*>(a.zeros.data) + row * a.zeros.stride[0] * size;
    }
  }
  // A slab's first column: of whole groups that leave the last slab short, that one is the row's last 128 columns, less the
  // groups that the slab before had.
  __device__ __forceinline__ int from(int slab) const { return kFast && kPerSlab > 1 ? min(slab * kSlab, in_dim - kSlab) : slab * kSlab; }
  // Pull a slab's codes towards L2.
  __device__ __forceinline__ void prefetch(int slab) const {
    if (kFast && slab < slabs)
#pragma unroll
      for (int r = 0; r < 2; ++r) asm volatile("prefetch.global.L2 [%0];" ::"l"(code[r] + from(slab) / 2));
  }
  __device__ __forceinline__ void fetch(int slab, Slab& to) const {
    if (slab >= slabs) return;
    const int begin = from(slab);
    if constexpr (kFast) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < kPerSlab; ++c) {
          const uint8_t* at = code[r] + begin / 2 + c * (kGroup / 2);
          if constexpr (kWords == 1) {
            to.code[r][c][0] = __ldcs(reinterpret_cast<const unsigned int*>(at));
          } else if constexpr (kWords == 2) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(at));
            to.code[r][c][0] = v.x;
            to.code[r][c][1] = v.y;
          } else {
            const uint4 v = __ldcs(reinterpret_cast<const uint4*>(at));
            to.code[r][c][0] = v.x;
            to.code[r][c][1] = v.y;
            to.code[r][c][2] = v.z;
            to.code[r][c][3] = v.w;
          }
          to.scale[r][c] = *reinterpret_cast<const uint16_t*>(scale[r] + 2 * (begin / kGroup + c));
          if (kZeros) to.zero[r][c] = *reinterpret_cast<const uint16_t*>(zero[r] + 2 * (begin / kGroup + c));
        }
    } else {
      const int bytes = (in_dim + 1) / 2;
      const uint8_t* data = static_cast<const uint8_t*>(a.codes.data);
      const uint8_t* end = data + (a.out_dim - 1) * a.codes.stride[0] + bytes;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // a neighbour row's bytes do no harm: they are shifted out, or meet zeros of x
        const bool inside = a.codes.stride[1] == 1 && a.codes.stride[0] >= 0 && code[r] + begin / 2 - off[r] >= data &&
                            code[r] + begin / 2 + kSlab / 2 + 4 <= end;
#pragma unroll
        for (int c = 0; c < kPerSlab; ++c) {
          const int at = begin / 2 + c * (kGroup / 2) + 4 * kWords * t - off[r];
          const int group = begin / kGroup + c;
          const bool there = group * kGroup < in_dim;  // past the row, x is 0
          if (inside) {
#pragma unroll
            for (int w = 0; w <= kWords; ++w) to.code[r][c][w] = *reinterpret_cast<const uint32_t*>(code[r] + at + 4 * w);
          } else {
#pragma unroll
            for (int w = 0; w <= kWords; ++w) to.code[r][c][w] = edge_word(code[r], a.codes.stride[1], at + 4 * w, bytes);
          }
          to.scale[r][c] = there ? bits(scale[r] + group * a.scales.stride[1] * size, type) : 0u;
          if (kZeros) to.zero[r][c] = there ? bits(zero[r] + group * a.zeros.stride[1] * size, type) : 0u;
        }
      }
    }
  }
  __device__ __forceinline__ uint32_t word(const Slab& s, int r, int c, int w) const {
    return kFast ? s.code[r][c][w] : __funnelshift_r(s.code[r][c][w], s.code[r][c][kFast ? w : w + 1], 8 * off[r]);
  }
};

// acc += scale (products - shift sums): the sums of one group, of a thread's 2 x 2 results.
template <bool kZeros>
__device__ __forceinline__ void join(float (&acc)[4], const float (&d)[4], const float (&sums)[4], float s0, float s1, float z0,
                                     float z1) {
  acc[0] = fmaf(s0, kZeros ? fmaf(-z0, sums[0], d[0]) : d[0], acc[0]);
  acc[1] = fmaf(s0, kZeros ? fmaf(-z0, sums[1], d[1]) : d[1], acc[1]);
  acc[2] = fmaf(s1, kZeros ? fmaf(-z1, sums[0], d[2]) : d[2], acc[2]);
  acc[3] = fmaf(s1, kZeros ? fmaf(-z1, sums[1], d[3]) : d[3], acc[3]);
}

// 8 columns of a row of x, from column c on; 0 past the row. `units`: rows start on 16 bytes.
template <typename T> __device__ __noinline__ uint4 x_careful(const m3_w4_args& a, const T* row, int c) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (a.x.stride[1] == 1) {
    row_words<4>(reinterpret_cast<const uint8_t*>(row), 1, 2 * (int64_t)c, 2 * a.in_dim, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < a.in_dim)
        w[e >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(row + (c + e) * a.x.stride[1]) << (16 * (e & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ uint4 x_unit(const m3_w4_args& a, const T* row, int c, bool units) {
  return units && c + 8 <= a.in_dim ? *reinterpret_cast<const uint4*>(row + c) : x_careful(a, row, c);
}

__host__ __device__ __forceinline__ bool x_in_units(const m3_w4_args& a) {
  return a.x.stride[1] == 1 && (a.rows == 1 || a.x.stride[0] % 8 == 0) && (reinterpret_cast<uintptr_t>(a.x.data) & 15) == 0;
}

// The definition of one output, for sums that are not finite. NaN ends it: nothing else follows from there.
template <typename T> __device__ __noinline__ float by_definition(const m3_w4_args& a, int64_t row, int64_t out) {
  const int type = a.scales.dtype, size = type == M3_F32 ? 4 : 2;
  const T* x = static_cast<const T*>(a.x.data) + row * a.x.stride[0];
  const uint8_t* codes = static_cast<const uint8_t*>(a.codes.data) + out * a.codes.stride[0];
  auto at = [&](const m3_tensor& t, int64_t g) {
    return widen(bits(static_cast<const uint8_t*>(t.data) + (out * t.stride[0] + g * t.stride[1]) * size, type), type);
  };
  float sum = 0.0f;
  for (int64_t g = 0; g * a.group < a.in_dim && sum == sum; ++g) {
    const float scale = at(a.scales, g), zero = a.zeros.data ? at(a.zeros, g) : 8.0f;
    const int64_t first = g * a.group, last = min(a.in_dim, first + a.group);
#pragma unroll 4
    for (int64_t i = first; i < last; ++i) {
      const int code = codes[(i >> 1) * a.codes.stride[1]] >> (i & 1 ? 4 : 0) & 15;
      sum = fmaf(to_f(x[i * a.x.stride[1]]), scale * ((float)code - zero), sum);
    }
  }
  return sum;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// ---- up to 8 rows --------------------------------------------------------------------------------
// A stream of codes: one CTA for 16 outputs, its warps share the columns out, slab by slab, and meet in shared memory.
// x, a few KB, comes from L1 as the products want it. 10768 x 2560, groups of 128: 6.3 us at one row (2.2 TB/s of codes),
// 7.1 at eight, groups of 64 and 32: 7.7 and 9.5: one wave of CTAs, twenty warps an SM, whose time is the launch, the
// first codes and the meeting of the warps. 8192 x 8192: 17.8, 512 CTAs of sixteen warps, of which the registers allow
// one an SM, so four waves, each warp waiting for its two slabs of codes and for x (five of nine clocks a warp between
// instructions; 40 % of the issue slots, DRAM's rate to 21 %). Scales widened where they are fetched cost 1.6 us of 8.
// Rows of codes that are no whole words (10768 x 2561): 21.
constexpr int kMostWarps = 16;

template <typename T, int kWords, bool kFast, bool kZeros>
__global__ void __launch_bounds__(32 * kMostWarps) w4_few_kernel(const __grid_constant__ m3_w4_args a) {
  using W = Weight<T, kWords, kFast, kZeros>;
  constexpr int kAhead = 2;  // slabs whose codes are under way
  __shared__ float part[kMostWarps][8][16];
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int64_t o0 = (int64_t)blockIdx.x * 16;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const W weight(a, o0, lane);
  // Launched as a programmatic dependent: what the kernel before wrote, the weight too if it did, is there only after
  // the wait. Until then the first codes are pulled towards L2.
  for (int i = 0; i < kAhead; ++i) weight.prefetch(warp + i * warps);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool units = x_in_units(a);
  // (a thread's type of scales: 16 bits in the fast form)
  auto value = [&](uint32_t v) {
    if constexpr (!kFast) return widen(v, weight.type);
    return weight.type == M3_BF16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half((uint16_t)v));
  };
  // (past the last row: the last one again, not written)
  const T* row = static_cast<const T*>(a.x.data) + min(g, (int)a.rows - 1) * a.x.stride[0];
  typename W::Slab held[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) weight.fetch(warp + i * warps, held[i]);
  const uint32_t one2 = std::is_same<T, __half>::value ? 0x3C003C00u : 0x3F803F80u;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int slab0 = warp; slab0 < weight.slabs; slab0 += kAhead * warps) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int slab = slab0 + i * warps;
      if (slab >= weight.slabs) break;
      uint4 x[4];
      const int begin = weight.from(slab);
      const T* columns = row + begin + 8 * kWords * t;  // of word w: group w / kWords of the slab
      if (kFast) {
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] = *reinterpret_cast<const uint4*>(columns + w / kWords * W::kGroup + 8 * (w % kWords));
      } else if (a.x.stride[1] == 1 && begin >= 2 && begin + kSlab + 2 <= weight.in_dim) {
        const int off = (int)(reinterpret_cast<uintptr_t>(columns) & 3);
        uint32_t v[4][5];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint8_t* at = reinterpret_cast<const uint8_t*>(columns + w / kWords * W::kGroup + 8 * (w % kWords)) - off;
#pragma unroll
          for (int e = 0; e < 5; ++e) v[w][e] = reinterpret_cast<const uint32_t*>(at)[e];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w)
          x[w] = make_uint4(__funnelshift_r(v[w][0], v[w][1], 8 * off), __funnelshift_r(v[w][1], v[w][2], 8 * off),
                            __funnelshift_r(v[w][2], v[w][3], 8 * off), __funnelshift_r(v[w][3], v[w][4], 8 * off));
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] = x_unit(a, row, begin + w / kWords * W::kGroup + 8 * (kWords * t + w % kWords), units);
      }
#pragma unroll
      for (int c = 0; c < W::kPerSlab; ++c) {
        if (kFast && W::kPerSlab > 1 && begin + c * W::kGroup < slab * kSlab) continue;  // the slab before had it
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          uint32_t low[4], high[4];
          open8<T>(weight.word(held[i], 0, c, w), low);
          open8<T>(weight.word(held[i], 1, c, w), high);
          const uint4 b = x[c * kWords + w];
          mma<T>(d, low[0], high[0], low[1], high[1], b.x, b.y);
          mma<T>(d, low[2], high[2], low[3], high[3], b.z, b.w);
          if (kZeros) {
            mma<T>(sums, one2, one2, one2, one2, b.x, b.y);
            mma<T>(sums, one2, one2, one2, one2, b.z, b.w);
          }
        }
        constexpr int kZ = kZeros ? 1 : 0;
        join<kZeros>(acc, d, sums, value(held[i].scale[0][c]), value(held[i].scale[1][c]), value(held[i].zero[0][kZ * c]) - 8.0f,
                     value(held[i].zero[1][kZ * c]) - 8.0f);
      }
      weight.fetch(slab + kAhead * warps, held[i]);
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
    if (!finite(v)) v = by_definition<T>(a, r, out);
    yp[r * a.y.stride[0] + out * a.y.stride[1]] = from_f<T>(v);
  }
}

// ---- more rows -----------------------------------------------------------------------------------
// The products of more rows are the fifth-generation tensor cores' (the warp-level instruction takes about 27 clocks
// for 16 x 8 x 16 here: 21 us for the 10768 x 2560 weight at 64 rows). One CTA for 128 outputs and up to kN rows. TMA
// brings the codes and x, 64 columns a stage; three teams of four warps take the stages in turn and turn the codes into
// 16-bit values code - 8 in shared memory (exact), a thread an output; one warp issues the MMAs, which sum one group
// into one of four accumulators in tensor memory (and with zero points the sums of x beside it, by products with ones);
// four warps read it, a thread an output, and add it, scaled, to sums in registers, in float32. Where the outputs are
// too few for the SMs, a cluster of CTAs shares the columns out and its partial sums meet through distributed shared
// memory.
// What bounds it is the chain of waits, issue and commits of the MMA warp, about 0.25 us a stage, with 85 CTAs for 148
// SMs: 10768 x 2560, groups of 128, takes 14.2, 15.8 and 16.7 us at 16, 32 and 64 rows (20 with zero points, 26 in
// groups of 32), 47 at 256; 2560 x 5120 takes 12 at 64. Before the issuing warps went in step (one lane in a branch of
// its own sends addresses and descriptors through vector registers) 64 rows took 24; stages of 128 columns took 19.5
// against 17.9 then; the warp-level instruction took 15.3, 19.8 and 31 at 16, 32 and 64 rows.
constexpr int kManyOuts = 128, kStage = 64;  // outputs of a CTA, columns of a stage
constexpr int kStages = 4, kRing = 8;        // of codes as 16-bit values; of codes and x as they come (powers of two)
constexpr int kTeams = 3, kProducers = 128 * kTeams;
constexpr int kSumsRing = 4;

template <int kN> struct Many {
  static constexpr int kCols = kN < 32 ? kN : 32, kConsumers = 4 * (kN / kCols);  // columns of a thread's sums; warps
  static constexpr int kThreads = kProducers + 64 + 32 * kConsumers;
  static constexpr uint32_t kA = kManyOuts * kStage * 2, kX = kN * kStage * 2, kCodes = kManyOuts * kStage / 2;
  static constexpr uint32_t kOffX = kStages * kA, kOffCodes = kOffX + kRing * kX, kOffBars = kOffCodes + kRing * kCodes;
  static constexpr uint32_t kOffOnes = kOffBars + 1024;  // a tile of ones, with zero points only
  static constexpr uint32_t kBytes = 1024 + std::max<uint32_t>(kOffOnes, kN * kManyOuts * 4);  // without the ones
  static constexpr int kColumns = 2 * kSumsRing * kN;  // of tensor memory: products, and sums of x where there are zero points
};

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Whether the barrier's phase is over, without waiting.
__device__ __forceinline__ bool passed(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ void mma_if(uint32_t leader, uint32_t to, uint64_t da, uint64_t db, uint32_t id, uint32_t adds) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(to),
      "l"(da), "l"(db), "r"(id), "r"(adds), "r"(leader));
}
__device__ __forceinline__ uint32_t elect() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader;
}
__device__ __forceinline__ void expect_if(uint32_t leader, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}\n" ::"r"(bar),
      "r"(bytes), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void copy_if(uint32_t leader, uint32_t to, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}\n" ::"r"(
          to),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
      "r"(leader)
      : "memory");
}

// Columns of tensor memory from `from` on, this thread's row of them.
__device__ __forceinline__ void load(uint32_t from, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(from));
}
__device__ __forceinline__ void load(uint32_t from, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(from));
}

template <typename T, int kN, bool kZeros>
__global__ void __launch_bounds__(Many<kN>::kThreads, 1)
    w4_many_kernel(const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap x_map,
                   const __grid_constant__ m3_w4_args a, int split, bool code_tiles, bool x_tiles) {
  using M = Many<kN>;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (umma::smem_u32(raw) + 1023u) & ~1023u;
  uint8_t* smem = raw + (base - umma::smem_u32(raw));
  const uint32_t bars = base + M::kOffBars;
  auto full = [&](int s) { return bars + 8u * (s & (kStages - 1)); };
  auto sums_full = [&](int g) { return bars + 8u * (kStages + (g & (kSumsRing - 1))); };
  auto sums_empty = [&](int g) { return bars + 8u * (kStages + kSumsRing + (g & (kSumsRing - 1))); };
  auto came = [&](int s) { return bars + 8u * (kStages + 2 * kSumsRing + (s & (kRing - 1))); };
  auto freed = [&](int s) { return bars + 8u * (kStages + 2 * kSumsRing + kRing + (s & (kRing - 1))); };
  const uint32_t drained = bars + 8u * (kStages + 2 * kSumsRing + 2 * kRing), slot = drained + 8u;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  int rank = 0;
  if (split > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int64_t o0 = (int64_t)(blockIdx.x / split) * kManyOuts;
  const int64_t rows0 = (int64_t)blockIdx.y * kN;
  const int rows = (int)min((int64_t)kN, a.rows - rows0);
  const int in_dim = (int)a.in_dim;
  // this CTA's columns, whole slabs of 128
  const int slabs = (in_dim + kSlab - 1) / kSlab, per = (slabs + split - 1) / split;
  const int first = min(in_dim, rank * per * kSlab), last = min(in_dim, (rank + 1) * per * kSlab);
  const int stages = (last - first + kStage - 1) / kStage, groups = (last - first + a.group - 1) / a.group;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full(i)), "r"(4));
    for (int i = 0; i < kRing; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(came(i)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(freed(i)));
    }
    for (int i = 0; i < kSumsRing; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(sums_full(i)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sums_empty(i)), "r"(M::kConsumers));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(drained));
    asm volatile("fence.mbarrier_init.release.cluster;");
  }
  if (warp == kProducers / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(M::kColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    // Only now: the block of a kernel after this one, which waits for this one's end, could otherwise come to this SM
    // and take the columns first, and both would wait for good.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  // Launched as a programmatic dependent: what the kernel before wrote, the weight too if it did, is there only after
  // the wait.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool units = x_in_units(a);
  const T* xp = static_cast<const T*>(a.x.data) + rows0 * a.x.stride[0];
  if (kZeros) {
    const uint32_t one2 = std::is_same<T, __half>::value ? 0x3C003C00u : 0x3F803F80u;
    for (int i = tid; i < (int)M::kA / 16; i += M::kThreads)
      asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(base + M::kOffOnes + 16 * i), "r"(one2) : "memory");
    umma::fence_async_smem();
  }
  umma::fence_before();
  __syncthreads();
  umma::fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  float acc[M::kCols];  // the consumers' sums

  if (tid < kProducers) {
    // the teams take stages in turn; a thread's part of one is the 64 columns of an output
    const int out = tid & 127, team = warp >> 2, flip = (out >> 2) & 1;  // (the copy's 32-byte swizzle: halves change places every four rows)
    const uint8_t* data = static_cast<const uint8_t*>(a.codes.data);
    const uint8_t* codes = data + min(o0 + out, a.out_dim - 1) * a.codes.stride[0];
    const int bytes = (in_dim + 1) / 2;
    // Rows of bytes that no copy engine reads (not a multiple of 16 bytes apart) come as aligned words, nine a row and
    // stage, the team's threads along the rows, a turn ahead in registers; shared memory hands each thread its row.
    const bool staged = !code_tiles && a.codes.stride[1] == 1 && a.codes.stride[0] >= 0;
    const uint8_t* end = data + (a.out_dim - 1) * a.codes.stride[0] + bytes;
    const uint32_t staging = base + M::kOffCodes + team * (kManyOuts * 36);
    uint32_t ahead[9];
    auto fetch_rows = [&](int s) {
#pragma unroll
      for (int j = 0; j < 9; ++j) {
        const int i = 128 * j + out;
        const uint8_t* from = data + min(o0 + i / 9, a.out_dim - 1) * a.codes.stride[0] + (first + s * kStage) / 2;
        from += 4 * (i % 9) - (int)(reinterpret_cast<uintptr_t>(from) & 3);
        if (from >= data && from + 4 <= end) {
          ahead[j] = *reinterpret_cast<const uint32_t*>(from);
        } else {
          uint32_t v = 0;
          for (int b = 0; b < 4; ++b)
            if (from + b >= data && from + b < end) v |= (uint32_t)from[b] << (8 * b);
          ahead[j] = v;
        }
      }
    };
    if (staged && team < stages) fetch_rows(team);
    bool ok = true;
    for (int s = team; s < stages; s += kTeams) {
      uint32_t words[8];
      uint4 held[kN / 16];
      const int c0 = first + s * kStage;
      if (!x_tiles) {
        if (a.x.stride[1] == 1 && c0 >= 2 && c0 + kStage + 2 <= in_dim) {  // rows past the last: the last, not written
          uint32_t w[kN / 16][5];
          int off[kN / 16];
#pragma unroll
          for (int i = 0; i < kN / 16; ++i) {
            const T* from = xp + min((out >> 3) + 16 * i, rows - 1) * a.x.stride[0] + c0 + 8 * (out & 7);
            off[i] = (int)(reinterpret_cast<uintptr_t>(from) & 3);
            const uint32_t* aligned = reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(from) - off[i]);
#pragma unroll
            for (int e = 0; e < 5; ++e) w[i][e] = aligned[e];
          }
#pragma unroll
          for (int i = 0; i < kN / 16; ++i)
            held[i] = make_uint4(__funnelshift_r(w[i][0], w[i][1], 8 * off[i]), __funnelshift_r(w[i][1], w[i][2], 8 * off[i]),
                                 __funnelshift_r(w[i][2], w[i][3], 8 * off[i]), __funnelshift_r(w[i][3], w[i][4], 8 * off[i]));
        } else {
#pragma unroll
          for (int i = 0; i < kN / 16; ++i) {
            const int n = (out >> 3) + 16 * i, c = c0 + 8 * (out & 7);
            held[i] = make_uint4(0u, 0u, 0u, 0u);
            if (n < rows && c < in_dim) held[i] = x_unit(a, xp + n * a.x.stride[0], c, units);
          }
        }
      }
      if (ok) ok = umma::mbar_wait(came(s), (uint32_t)(s / kRing) & 1u);
      if (code_tiles) {
        const uint32_t from = base + M::kOffCodes + (s & (kRing - 1)) * M::kCodes + out * 32;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(words[4 * h]), "=r"(words[4 * h + 1]), "=r"(words[4 * h + 2]), "=r"(words[4 * h + 3])
                       : "r"(from + ((h ^ flip) << 4))
                       : "memory");
      } else if (staged) {
        asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory");  // the team has read what this one replaces
#pragma unroll
        for (int j = 0; j < 9; ++j) asm volatile("st.shared.u32 [%0], %1;" ::"r"(staging + 4 * (128 * j + out)), "r"(ahead[j]) : "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + team) : "memory");
        if (s + kTeams < stages) fetch_rows(s + kTeams);
        const int off = (int)(reinterpret_cast<uintptr_t>(codes + c0 / 2) & 3);
        uint32_t w[9];
#pragma unroll
        for (int j = 0; j < 9; ++j) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[j]) : "r"(staging + 36 * out + 4 * j) : "memory");
#pragma unroll
        for (int j = 0; j < 8; ++j) words[j] = __funnelshift_r(w[j], w[j + 1], 8 * off);
      } else {
        row_words<8>(codes, a.codes.stride[1], c0 / 2, bytes, words);
      }
      // the MMAs of stage s - kStages are done with what this one replaces
      if (s >= kStages && ok) ok = umma::mbar_wait(freed(s - kStages), (uint32_t)((s - kStages) / kRing) & 1u);
      if (!x_tiles)
#pragma unroll
        for (int i = 0; i < kN / 16; ++i) {
          const int n = (out >> 3) + 16 * i;
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + M::kOffX + (s & (kRing - 1)) * M::kX + n * 128 +
                                                                        (((out ^ n) & 7) << 4)),
                       "r"(held[i].x), "r"(held[i].y), "r"(held[i].z), "r"(held[i].w)
                       : "memory");
        }
      const uint32_t to = base + (s & (kStages - 1)) * M::kA + out * 128;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        uint32_t v[4];
        open8<T>(words[w], v);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + ((w ^ (out & 7)) << 4)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                     "r"(v[3])
                     : "memory");
      }
      umma::fence_async_smem();
      __syncwarp();
      if (lane == 0) arrive(full(s));  // one arrival a warp: a barrier takes them one by one
    }
  } else if (warp == kProducers / 32 + 1) {
    // The copies; a stage's barrier completes without bytes where TMA cannot read either. A stage that the MMAs are done
    // with has been read by the teams too. (In step, as the warp of the MMAs: one lane took 0.3 us a stage.)
    const uint32_t leader = elect();
    const uint32_t bytes = (code_tiles ? M::kCodes : 0) + (x_tiles ? M::kX : 0);
    bool ok = true;
    int s = 0;
    for (; s < stages; ++s) {
      if (s >= kRing) {
        ok = __all_sync(0xffffffffu, umma::mbar_wait(freed(s), (uint32_t)(s / kRing - 1) & 1u));
        if (!ok) break;
      }
      expect_if(leader, came(s), bytes);
      const int c = first + s * kStage;
      if (code_tiles) copy_if(leader, base + M::kOffCodes + (s & (kRing - 1)) * M::kCodes, &code_map, c / 2, (int)o0, came(s));
      if (x_tiles) copy_if(leader, base + M::kOffX + (s & (kRing - 1)) * M::kX, &x_map, c, (int)rows0, came(s));
    }
    if (!ok)  // gave up: the copies under way land before the block's shared memory goes
      for (int i = max(0, s - kRing); i < s; ++i) umma::mbar_wait(came(i), (uint32_t)(i / kRing) & 1u);
  } else if (warp == kProducers / 32) {
    // The chain that all else waits for: no division, one commit a stage and one a group. The whole warp goes through
    // it and one lane's instructions count, so that addresses and descriptors are the warp's, in uniform registers.
    const uint32_t leader = elect();
    const uint32_t id = umma::idesc(kManyOuts, kN, std::is_same<T, __nv_bfloat16>::value, false, false);
    const uint32_t acc0 = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t da0 = umma::sdesc(base, 16, 1024), db0 = umma::sdesc(base + M::kOffX, 16, 1024);
    const uint64_t ones = umma::sdesc(base + M::kOffOnes, 16, 1024);
    auto product = [&](uint32_t to, uint64_t da, uint64_t db, uint32_t adds) {
      mma_if(leader, to, da, db, id, adds);
      if (kZeros) mma_if(leader, to + kSumsRing * kN, ones, db, id, adds);  // the sums of x, the same for every output
    };
    // A stage is half a group, a group or two; columns past the row are zeros of x.
    const int parts = a.group == 32 ? 2 : 1, stages_of = a.group == 128 ? 2 : 1;
    auto empty = [&](int g) { return g < kSumsRing || g >= groups || passed(sums_empty(g), (uint32_t)(g / kSumsRing - 1) & 1u); };
    auto begin = [&](int g) { return g < kSumsRing || umma::mbar_wait(sums_empty(g), (uint32_t)(g / kSumsRing - 1) & 1u); };
    bool ok = true, come = false, room = true;  // the stage's operands, its group's accumulator: looked at a stage ahead
    int g = 0;
    for (int s = 0; s < stages && ok; ++s) {
      const bool opens = stages_of == 1 || (s & 1) == 0, closes = stages_of == 1 || (s & 1) == 1 || s + 1 == stages;
      if (!__all_sync(0xffffffffu, come && room)) {
        ok = umma::mbar_wait(full(s), (uint32_t)(s / kStages) & 1u);
        if (opens) ok = ok && begin(g);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      umma::fence_after();
      come = s + 1 < stages && passed(full(s + 1), (uint32_t)((s + 1) / kStages) & 1u);
      room = closes ? empty(g + parts) : true;
      const uint64_t da = umma::sdesc_at(da0, (s & (kStages - 1)) * M::kA), db = umma::sdesc_at(db0, (s & (kRing - 1)) * M::kX);
      uint32_t to = acc0 + (g & (kSumsRing - 1)) * kN;
      product(to, da, db, !opens);
      product(to, umma::sdesc_at(da, 32), umma::sdesc_at(db, 32), 1);
      if (parts == 2) {
        commit_if(leader, sums_full(g));
        if (++g == groups) {
          commit_if(leader, freed(s));
          break;
        }
        ok = __all_sync(0xffffffffu, begin(g));
        if (!ok) break;
        umma::fence_after();
        to = acc0 + (g & (kSumsRing - 1)) * kN;
      }
      product(to, umma::sdesc_at(da, 64), umma::sdesc_at(db, 64), parts == 1);
      product(to, umma::sdesc_at(da, 96), umma::sdesc_at(db, 96), 1);
      if (closes) commit_if(leader, sums_full(g++));
      commit_if(leader, freed(s));
    }
    commit_if(leader, drained);  // the MMAs end, and their arrivals, before their memory is given back
    umma::mbar_wait(drained, 0);
  } else {
    const int quarter = warp & 3, out = quarter * 32 + lane, col0 = M::kCols * ((warp - kProducers / 32 - 2) >> 2);
    const int64_t o = min(o0 + out, a.out_dim - 1);
#pragma unroll
    for (int n = 0; n < M::kCols; ++n) acc[n] = 0.0f;
    const int type = a.scales.dtype, size = type == M3_F32 ? 4 : 2;
    auto start = [&](const m3_tensor& t) {
      return static_cast<const uint8_t*>(t.data) + (o * t.stride[0] + first / a.group * t.stride[1]) * size;
    };
    auto fetch = [&](const uint8_t*& at, int64_t stride, int g) {
      const uint32_t v = g < groups ? bits(at, type) : 0u;
      at += stride * size;
      return v;
    };
    auto value = [&](uint32_t v) { return widen(v, type); };
    const uint8_t *scale_at = start(a.scales), *zero_at = kZeros ? start(a.zeros) : nullptr;
    constexpr int kPart = kZeros ? 8 : 16;  // columns read at a time
    constexpr int kAhead = kZeros ? 2 : 4;  // groups whose scales are under way
    uint32_t s_held[kAhead], z_held[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      s_held[i] = fetch(scale_at, a.scales.stride[1], i);
      z_held[i] = kZeros ? fetch(zero_at, a.zeros.stride[1], i) : 0u;
    }
    bool ok = true;
    for (int g0 = 0; g0 < groups && ok; g0 += kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int g = g0 + i;
        if (g >= groups) break;
        const float s = value(s_held[i]), z = value(z_held[i]) - 8.0f;
        s_held[i] = fetch(scale_at, a.scales.stride[1], g + kAhead);
        if (kZeros) z_held[i] = fetch(zero_at, a.zeros.stride[1], g + kAhead);
        ok = __all_sync(0xffffffffu, umma::mbar_wait(sums_full(g), (uint32_t)(g / kSumsRing) & 1u));
        if (!ok) break;
        umma::fence_after();
        const uint32_t from = tmem + (g & (kSumsRing - 1)) * kN + col0 + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
        for (int n0 = 0; n0 < M::kCols; n0 += kPart) {
          uint32_t r[kPart], u[kPart];
          load(from + n0, r);
          if (kZeros) load(from + kSumsRing * kN + n0, u);
          umma::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < kPart; ++e) {
            const float d = __uint_as_float(r[e]);
            acc[n0 + e] = fmaf(s, kZeros ? fmaf(-z, __uint_as_float(u[e]), d) : d, acc[n0 + e]);
          }
        }
        umma::fence_before();
        __syncwarp();
        if (lane == 0) arrive(sums_empty(g));
      }
    }
  }
  __syncwarp();
  umma::fence_before();
  __syncthreads();
  umma::fence_after();
  if (warp == kProducers / 32)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(M::kColumns));
  T* yp = static_cast<T*>(a.y.data);
  const int out = (warp & 3) * 32 + lane;
  const bool consumer = warp > kProducers / 32 + 1;
  const int col0 = consumer ? M::kCols * ((warp - kProducers / 32 - 2) >> 2) : 0;
  if (split == 1) {
    if (consumer && o0 + out < a.out_dim) {
      uint32_t again = 0;
#pragma unroll
      for (int n = 0; n < M::kCols; ++n) {
        if (col0 + n >= rows) continue;
        yp[(rows0 + col0 + n) * a.y.stride[0] + (o0 + out) * a.y.stride[1]] = from_f<T>(acc[n]);
        again |= finite(acc[n]) ? 0u : 1u << n;
      }
      for (; again; again &= again - 1) {
        const int64_t row = rows0 + col0 + __ffs(again) - 1;
        yp[row * a.y.stride[0] + (o0 + out) * a.y.stride[1]] = from_f<T>(by_definition<T>(a, row, o0 + out));
      }
    }
    return;
  }
  // the cluster's partial sums: [kN][128] in every CTA's shared memory; CTA r adds up rows r kN / split ...
  float* part = reinterpret_cast<float*>(smem);
  if (consumer) {
#pragma unroll
    for (int n = 0; n < M::kCols; ++n) part[(col0 + n) * kManyOuts + out] = acc[n];
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int share = kN / split;
  for (int i = tid; i < share * kManyOuts; i += M::kThreads) {
    const int n = rank * share + i / kManyOuts, oo = i % kManyOuts;
    float v = 0.0f;
    for (int r = 0; r < split; ++r) {
      uint32_t at;
      float p;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(umma::smem_u32(part + n * kManyOuts + oo)), "r"(r));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(p) : "r"(at) : "memory");
      v += p;
    }
    if (n >= rows || o0 + oo >= a.out_dim) continue;
    if (!finite(v)) v = by_definition<T>(a, rows0 + n, o0 + oo);
    yp[(rows0 + n) * a.y.stride[0] + (o0 + oo) * a.y.stride[1]] = from_f<T>(v);
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // no CTA leaves while another reads its sums
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
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

// Boxes of box_cols x box_rows of a matrix; what lies outside reads as 0.
bool encode(CUtensorMap* map, CUtensorMapDataType type, const m3_tensor& t, int64_t cols, int64_t rows, int elem, int box_cols,
            int box_rows, CUtensorMapSwizzle swizzle) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(rows == 1 ? (cols * elem + 15) / 16 * 16 : t.stride[0] * elem)};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, step[2] = {1, 1};
  return enc(map, type, 2, t.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int kN, bool kZeros> cudaError_t launch_many(const m3_w4_args& a, cudaStream_t stream) {
  // CTAs for the columns of 128 outputs: while that leaves SMs idle and each has four slabs or more
  const int64_t tiles = (a.out_dim + kManyOuts - 1) / kManyOuts, slabs = (a.in_dim + kSlab - 1) / kSlab;
  const int64_t row_tiles = (a.rows + kN - 1) / kN;
  int split = 1;
  while (split < 8 && 2 * split * tiles * row_tiles <= sm_count() && slabs >= 8 * split) split *= 2;
  const size_t smem = Many<kN>::kBytes + (kZeros ? Many<kN>::kA : 0);
  auto kernel = w4_many_kernel<T, kN, kZeros>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config(dim3((unsigned)(tiles * split), (unsigned)row_tiles), Many<kN>::kThreads, smem, stream, attr);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = split > 1 ? 2 : 1;
  const bool code_tiles = a.codes.stride[1] == 1 && (a.codes.stride[0] > 0 || a.out_dim == 1) && a.codes.stride[0] % 16 == 0 &&
                          reinterpret_cast<uintptr_t>(a.codes.data) % 16 == 0;
  const bool x_tiles = x_in_units(a) && a.x.stride[0] > 0;
  CUtensorMap code_map = {}, x_map = {};
  if ((code_tiles && !encode(&code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, (a.in_dim + 1) / 2, a.out_dim, 1, kStage / 2,
                             kManyOuts, CU_TENSOR_MAP_SWIZZLE_32B)) ||
      (x_tiles && !encode(&x_map, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          a.x, a.in_dim, a.rows, 2, kStage, kN, CU_TENSOR_MAP_SWIZZLE_128B))) {
    return cudaErrorInvalidValue;
  }
  return cudaLaunchKernelEx(&cfg, kernel, code_map, x_map, a, split, code_tiles, x_tiles);
}

// Past 64 rows, the weight is read once for every 64.
template <typename T, bool kZeros> cudaError_t launch_many_rows(const m3_w4_args& a, cudaStream_t stream) {
  if (a.rows > 32) return launch_many<T, 64, kZeros>(a, stream);
  return a.rows > 16 ? launch_many<T, 32, kZeros>(a, stream) : launch_many<T, 16, kZeros>(a, stream);
}

template <typename T, int kWords, bool kFast, bool kZeros> cudaError_t launch_few(const m3_w4_args& a, cudaStream_t stream) {
  // warps for the columns of 16 outputs: enough to give every SM 16, while each has two slabs or more
  const int64_t tiles = (a.out_dim + 15) / 16, slabs = (a.in_dim + kSlab - 1) / kSlab;
  int warps = 4;
  while (warps < kMostWarps && tiles * warps < (int64_t)16 * sm_count() && 4 * warps <= slabs) warps *= 2;
  cudaLaunchAttribute chained;
  const cudaLaunchConfig_t cfg = config(dim3((unsigned)tiles), 32 * warps, 0, stream, &chained);
  return cudaLaunchKernelEx(&cfg, w4_few_kernel<T, kWords, kFast, kZeros>, a);
}

template <typename T, int kWords> cudaError_t launch_group(const m3_w4_args& a, cudaStream_t stream) {
  const bool fast = a.codes.stride[1] == 1 && a.codes.stride[0] % (4 * kWords) == 0 &&
                    reinterpret_cast<uintptr_t>(a.codes.data) % (4 * kWords) == 0 && a.scales.dtype != M3_F32 && x_in_units(a) &&
                    a.in_dim % a.group == 0 && a.in_dim >= kSlab && a.scales.stride[1] == 1 && (a.zeros.data == nullptr || a.zeros.stride[1] == 1);
  if (a.zeros.data) return fast ? launch_few<T, kWords, true, true>(a, stream) : launch_few<T, kWords, false, true>(a, stream);
  return fast ? launch_few<T, kWords, true, false>(a, stream) : launch_few<T, kWords, false, false>(a, stream);
}

template <typename T> cudaError_t launch_type(const m3_w4_args& a, cudaStream_t stream) {
  if (a.rows > 8) return a.zeros.data ? launch_many_rows<T, true>(a, stream) : launch_many_rows<T, false>(a, stream);
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
  constexpr int64_t kMost = INT32_MAX - 4096;  // columns a few stages past the row's end still count in 32 bits
  if (a.rows > 64 * 65535 || a.out_dim > kMost || a.in_dim > kMost)
    return report_error(M3_ERR_SHAPE, "m3_linear_w4: rows above 64 * 65535, or out_dim or in_dim above 2^31 - 4097");
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
