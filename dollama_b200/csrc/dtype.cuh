// Element types of the int8 language-model operators (dlm_dtype) and their conversions to and from
// the 32-bit floats that every sum, norm and softmax statistic is held in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace dlm {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// a * b + c in fp32 from two elements (the products of 16-bit elements are exact).
template <typename T>
__device__ __forceinline__ float fma_f(T a, T b, float c);
template <>
__device__ __forceinline__ float fma_f<float>(float a, float b, float c) { return fmaf(a, b, c); }
template <>
__device__ __forceinline__ float fma_f<__half>(__half a, __half b, float c) {
  float d;
  asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(__half_as_ushort(a)), "h"(__half_as_ushort(b)), "f"(c));
  return d;
}
template <>
__device__ __forceinline__ float fma_f<__nv_bfloat16>(__nv_bfloat16 a, __nv_bfloat16 b, float c) {
  float d;
  asm("fma.rn.f32.bf16 %0, %1, %2, %3;"
      : "=f"(d)
      : "h"(__bfloat16_as_ushort(a)), "h"(__bfloat16_as_ushort(b)), "f"(c));
  return d;
}

// N consecutive elements as one load or store of sizeof(T) * N <= 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// a[j] += b[j], rounded once to T
template <int N>
__device__ __forceinline__ void add_to(Vec<float, N>& a, const Vec<float, N>& b) {
#pragma unroll
  for (int j = 0; j < N; ++j) a.v[j] += b.v[j];
}
template <int N>
__device__ __forceinline__ void add_to(Vec<__half, N>& a, const Vec<__half, N>& b) {
  if constexpr (N == 1) {
    a.v[0] = __hadd(a.v[0], b.v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const __half2 s = __hadd2(__halves2half2(a.v[j], a.v[j + 1]), __halves2half2(b.v[j], b.v[j + 1]));
      a.v[j] = __low2half(s);
      a.v[j + 1] = __high2half(s);
    }
  }
}
template <int N>
__device__ __forceinline__ void add_to(Vec<__nv_bfloat16, N>& a, const Vec<__nv_bfloat16, N>& b) {
  if constexpr (N == 1) {
    a.v[0] = __hadd(a.v[0], b.v[0]);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const __nv_bfloat162 s = __hadd2(__halves2bfloat162(a.v[j], a.v[j + 1]), __halves2bfloat162(b.v[j], b.v[j + 1]));
      a.v[j] = __low2bfloat16(s);
      a.v[j + 1] = __high2bfloat16(s);
    }
  }
}

// max that keeps a NaN of either operand
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// max_j |x_j|, NaN if any is
template <int N>
__device__ __forceinline__ float max_abs(const Vec<float, N>& x, float m) {
#pragma unroll
  for (int j = 0; j < N; ++j) m = max_nan(m, fabsf(x.v[j]));
  return m;
}
template <int N>
__device__ __forceinline__ float max_abs(const Vec<__half, N>& x, float m) {
  __half2 t = __habs2(__halves2half2(x.v[0], x.v[1]));
#pragma unroll
  for (int j = 2; j < N; j += 2) t = __hmax2_nan(t, __habs2(__halves2half2(x.v[j], x.v[j + 1])));
  return max_nan(m, __half2float(__hmax_nan(__low2half(t), __high2half(t))));
}
template <int N>
__device__ __forceinline__ float max_abs(const Vec<__nv_bfloat16, N>& x, float m) {
  __nv_bfloat162 t = __habs2(__halves2bfloat162(x.v[0], x.v[1]));
#pragma unroll
  for (int j = 2; j < N; j += 2) t = __hmax2_nan(t, __habs2(__halves2bfloat162(x.v[j], x.v[j + 1])));
  return max_nan(m, __bfloat162float(__hmax_nan(__low2bfloat16(t), __high2bfloat16(t))));
}

// The absmax int8 codes round_half_away(127 x_j / a) of N values (a multiple of 4) of a row of
// largest magnitude a, given v_j = x_j * (127 / a) in fp32, which is within `err` of the quotient:
// away from a half-integer v_j rounds as the quotient does.  Next to one `exact(j)` forms the
// quotient in double (quant_exact), on a branch that few vectors take (two in 10^3 for eight values
// and err 2^-14).  Rounding is the addition of 3 * 2^22, whose sum's low byte is the code.
template <int N, typename F>
__device__ __forceinline__ void quant_codes(const float (&v)[N], float err, uint32_t (&out)[N / 4], F&& exact) {
  constexpr float kMagic = 12582912.0f;
  uint32_t t[N];
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float r = __fadd_rn(v[j], kMagic);
    t[j] = __float_as_uint(r);
    far = fmaxf(far, fabsf(__fsub_rn(v[j], __fsub_rn(r, kMagic))));
  }
  if (far >= 0.5f - err) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (fabsf(__fsub_rn(v[j], __fsub_rn(__uint_as_float(t[j]), kMagic))) >= 0.5f - err)
        t[j] = static_cast<uint32_t>(exact(j));
  }
#pragma unroll
  for (int j = 0; j < N; j += 4)
    out[j / 4] = __byte_perm(__byte_perm(t[j], t[j + 1], 0x0040), __byte_perm(t[j + 2], t[j + 3], 0x0040), 0x5410);
}

// The codes of N values x_j of a 16-bit type in a row of largest magnitude a, from v_j = x_j * r in fp32
// with r = (127 / a) (1 + 2^-21), without a check: with integers x = m 2^s, a = n 2^s (m < 2^11, as
// |x| <= a), the quotient 127 m / n is a half-integer or differs from every one by a fraction of at
// least 1 / (254 m) > 2^-19 of itself.  The three roundings of v_j move it by less than 2^-22, so the
// factor lies in (1, 1 + 2^-20): exact halves go away from zero, nothing else crosses one.
constexpr float kHalvesAway = 1.0f + 0x1p-21f;
template <int N>
__device__ __forceinline__ void quant_codes_16(const float (&v)[N], uint32_t (&out)[N / 4]) {
  uint32_t t[N];
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = __float_as_uint(__fadd_rn(v[j], 12582912.0f));
#pragma unroll
  for (int j = 0; j < N; j += 4)
    out[j / 4] = __byte_perm(__byte_perm(t[j], t[j + 1], 0x0040), __byte_perm(t[j + 2], t[j + 3], 0x0040), 0x5410);
}

// The same code from double: 127 x is exact for x of up to 46 bits, and the correctly rounded
// division returns an exact tie as one.
__device__ __forceinline__ int quant_exact(double x, double a) {
  return static_cast<int>(round(__ddiv_rn(__dmul_rn(127.0, x), a)));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
inline size_t dtype_size(int dtype) { return dtype == DLM_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == DLM_F32 || dtype == DLM_F16 || dtype == DLM_BF16; }

}  // namespace dlm

// Runs the given statements with T the element type of a valid dlm_dtype.
#define DLM_DISPATCH_DTYPE(dtype, T, ...)                \
  do {                                                   \
    if ((dtype) == DLM_F32) {                            \
      using T = float;                                   \
      __VA_ARGS__;                                       \
    } else if ((dtype) == DLM_F16) {                     \
      using T = __half;                                  \
      __VA_ARGS__;                                       \
    } else {                                             \
      using T = __nv_bfloat16;                           \
      __VA_ARGS__;                                       \
    }                                                    \
  } while (0)
