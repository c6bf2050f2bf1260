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

// N consecutive elements as one load or store of sizeof(T) * N <= 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// max that keeps a NaN of either operand
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The absmax int8 code of x in a row of largest magnitude a, round_half_away(127 x / a), given
// v = x * (127 / a) in fp32.  v is within 2^-15 of the quotient (three roundings of at most
// 127 * 2^-24 each), so away from a half-integer it rounds as the quotient does; next to one the
// quotient is formed in double, where 127 * x is exact for products of up to 46 bits and the
// correctly rounded division returns an exact tie as one.
__device__ __forceinline__ int quant_code(float v, double x, double a) {
  const int q = __float2int_rn(v);
  const float d = fabsf(v - static_cast<float>(q));
  if (d < 0.5f - 0x1p-13f) return q;
  return static_cast<int>(round(__ddiv_rn(__dmul_rn(127.0, x), a)));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
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
