// The int8 K/V cache of a language model: quantizing K and V rows as they are written, and reading
// them back.
//
// One row is the Dh values of one token and one head; its scale is a / 127 (a = largest magnitude)
// and its codes round_half_away(127 x / a), the rule of dlm_quantize_act_i8.  Codes are
// [B][H][Lmax][Dh], scales [B][H][Lmax], so a head's keys are contiguous for the attention that
// reads them.  A row is handled by Dh / 8 neighbouring lanes, 8 values each: reads of 16 or 32 bytes
// a lane, one shuffle tree for the largest magnitude, 8-byte code stores.  Memory-bound.
#include <cstdint>

#include "dtype.cuh"
#include "kv_i8.h"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kKvThreads = 256;

template <typename T>
struct Oct {  // 8 elements in 16-byte pieces
  static constexpr int kPieces = sizeof(T) / 2;
  Vec<T, 16 / sizeof(T)> v[kPieces];
  __device__ __forceinline__ T& at(int i) { return v[i / (16 / sizeof(T))].v[i % (16 / sizeof(T))]; }
};

// The cache row of (token b, s; head) and whether it exists: s below the sequence's count and its
// position inside the cache (a position outside raises the device status word).
__device__ __forceinline__ bool cache_row(const KvShape& p, int b, int s, int hd, size_t& row) {
  const int n = p.counts ? p.counts[b] : p.S;
  if (s >= n) return false;
  const long long at = static_cast<long long>(p.pos[b]) + s;
  if (at < 0 || at >= p.Lmax) {
    if (p.status) atomicCAS(p.status, 0, kDevBadPosition);
    return false;
  }
  row = (static_cast<size_t>(b) * p.H + hd) * p.Lmax + static_cast<size_t>(at);
  return true;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kKvThreads)
    kv_append_kernel(const T* __restrict__ k, long long ldk, const T* __restrict__ v, long long ldv,
                     int8_t* __restrict__ kq, float* __restrict__ ks, int8_t* __restrict__ vq,
                     float* __restrict__ vs, const KvShape p) {
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  constexpr int G = DH / 8;
  const long long u = (static_cast<long long>(blockIdx.x) * kKvThreads + threadIdx.x) / G;
  const int c = threadIdx.x % G;
  const long long rows = static_cast<long long>(p.B) * p.S * p.H;
  // unit u: K row u, then (from `rows` on) V row u - rows
  const bool is_v = u >= rows;
  const long long i = is_v ? u - rows : u;
  size_t row = 0;
  bool live = u < 2 * rows;
  int hd = 0;
  long long tok = 0;
  if (live) {
    hd = static_cast<int>(i % p.H);
    tok = i / p.H;
    live = cache_row(p, static_cast<int>(tok / p.S), static_cast<int>(tok % p.S), hd, row);
  }
  Oct<T> x;
  float a = 0.0f;
  if (live) {
    const T* src = (is_v ? v + tok * ldv : k + tok * ldk) + hd * DH + c * 8;
#pragma unroll
    for (int j = 0; j < Oct<T>::kPieces; ++j)
      x.v[j] = reinterpret_cast<const Vec<T, 16 / sizeof(T)>*>(src)[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max_nan(a, fabsf(to_f(x.at(j))));
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  if (!live) return;
  const bool finite = a < INFINITY;  // false for a NaN as well
  const bool tiny = a < 1e-30f;      // 127 / a may leave fp32's range: quotients in double
  const float rq = 127.0f / a;
  Vec<int8_t, 8> q;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = to_f(x.at(j));
    int code = 0;
    if (finite && a > 0.0f)
      code = tiny ? static_cast<int>(round(__ddiv_rn(127.0 * static_cast<double>(f), static_cast<double>(a))))
                  : quant_code(f * rq, static_cast<double>(f), static_cast<double>(a));
    q.v[j] = static_cast<int8_t>(code);
  }
  *reinterpret_cast<Vec<int8_t, 8>*>((is_v ? vq : kq) + row * DH + c * 8) = q;
  // a row that holds a NaN or an infinity: codes 0 under a NaN scale
  if (c == 0) (is_v ? vs : ks)[row] = finite ? __fdiv_rn(a, 127.0f) : NAN;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kKvThreads)
    kv_read_kernel(const int8_t* __restrict__ kq, const float* __restrict__ ks,
                   const int8_t* __restrict__ vq, const float* __restrict__ vs, T* __restrict__ k,
                   long long ldk, T* __restrict__ v, long long ldv, const KvShape p) {
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  constexpr int G = DH / 8;
  const long long u = (static_cast<long long>(blockIdx.x) * kKvThreads + threadIdx.x) / G;
  const int c = threadIdx.x % G;
  const long long rows = static_cast<long long>(p.B) * p.S * p.H;
  if (u >= 2 * rows) return;
  const bool is_v = u >= rows;
  const long long i = is_v ? u - rows : u;
  const int hd = static_cast<int>(i % p.H);
  const long long tok = i / p.H;
  size_t row;
  if (!cache_row(p, static_cast<int>(tok / p.S), static_cast<int>(tok % p.S), hd, row)) return;
  const float sc = (is_v ? vs : ks)[row];
  const Vec<int8_t, 8> q = *reinterpret_cast<const Vec<int8_t, 8>*>((is_v ? vq : kq) + row * DH + c * 8);
  Oct<T> x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x.at(j) = from_f<T>(static_cast<float>(q.v[j]) * sc);
  T* dst = (is_v ? v + tok * ldv : k + tok * ldk) + hd * DH + c * 8;
#pragma unroll
  for (int j = 0; j < Oct<T>::kPieces; ++j) reinterpret_cast<Vec<T, 16 / sizeof(T)>*>(dst)[j] = x.v[j];
}

int check(const char* fn, const void* k, int ldk, const void* v, int ldv, const void* kq, const void* ks,
          const void* vq, const void* vs, const KvShape& p, int Dh, int dtype) {
  DLM_REQUIRE(p.B >= 0 && p.S >= 0 && p.H >= 0 && p.Lmax >= 0, DLM_ERR_INVALID, "%s: negative size", fn);
  DLM_REQUIRE(dtype_ok(dtype), DLM_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  DLM_REQUIRE(Dh == 64 || Dh == 128, DLM_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128)", fn, Dh);
  if (p.B == 0 || p.S == 0 || p.H == 0 || p.Lmax == 0) return DLM_OK;
  DLM_REQUIRE(k && v && kq && ks && vq && vs && p.pos, DLM_ERR_INVALID, "%s: null pointer", fn);
  const long long width = static_cast<long long>(p.H) * Dh;
  DLM_REQUIRE(ldk >= width && ldv >= width, DLM_ERR_INVALID, "%s: a token stride is below H * Dh = %lld", fn,
              width);
  const int vec = static_cast<int>(16 / dtype_size(dtype));
  DLM_REQUIRE(aligned16(k) && aligned16(v) && ldk % vec == 0 && ldv % vec == 0, DLM_ERR_INVALID,
              "%s: k / v rows must start on 16-byte boundaries", fn);
  DLM_REQUIRE(aligned16(kq) && aligned16(vq), DLM_ERR_INVALID, "%s: cache codes must be 16-byte aligned", fn);
  DLM_REQUIRE(2ll * p.B * p.S * p.H * (Dh / 8) / kKvThreads < (1ll << 31) - 1, DLM_ERR_UNSUPPORTED,
              "%s: too many rows", fn);
  return DLM_OK;
}

unsigned grid_of(const KvShape& p, int Dh) {
  const long long threads = 2ll * p.B * p.S * p.H * (Dh / 8);
  return static_cast<unsigned>((threads + kKvThreads - 1) / kKvThreads);
}

}  // namespace

}  // namespace dlm

extern "C" {

int dlm_kv_i8_append(const void* k, int ldk, const void* v, int ldv, int8_t* kq, float* kscale, int8_t* vq,
                     float* vscale, int B, int S, int H, int Dh, int Lmax, const int* pos,
                     const int* counts, int dtype, void* stream) {
  using namespace dlm;
  KvShape p{B, S, H, Lmax, pos, counts, nullptr};
  const int rc = check("kv_i8_append", k, ldk, v, ldv, kq, kscale, vq, vscale, p, Dh, dtype);
  if (rc != DLM_OK || B == 0 || S == 0 || H == 0 || Lmax == 0) return rc;
  p.status = device_status_ptr();
  const dim3 grid(grid_of(p, Dh));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    const T* kt = static_cast<const T*>(k);
    const T* vt = static_cast<const T*>(v);
    if (Dh == 64)
      DLM_CHECK_CUDA(launch_pdl(kv_append_kernel<T, 64>, grid, dim3(kKvThreads), 0, s, kt, ldk, vt, ldv, kq,
                                kscale, vq, vscale, p));
    else
      DLM_CHECK_CUDA(launch_pdl(kv_append_kernel<T, 128>, grid, dim3(kKvThreads), 0, s, kt, ldk, vt, ldv, kq,
                                kscale, vq, vscale, p));
  });
  return DLM_OK;
}

int dlm_kv_i8_read(const int8_t* kq, const float* kscale, const int8_t* vq, const float* vscale, void* k,
                   int ldk, void* v, int ldv, int B, int S, int H, int Dh, int Lmax, const int* pos,
                   const int* counts, int dtype, void* stream) {
  using namespace dlm;
  KvShape p{B, S, H, Lmax, pos, counts, nullptr};
  const int rc = check("kv_i8_read", k, ldk, v, ldv, kq, kscale, vq, vscale, p, Dh, dtype);
  if (rc != DLM_OK || B == 0 || S == 0 || H == 0 || Lmax == 0) return rc;
  p.status = device_status_ptr();
  const dim3 grid(grid_of(p, Dh));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    T* kt = static_cast<T*>(k);
    T* vt = static_cast<T*>(v);
    if (Dh == 64)
      DLM_CHECK_CUDA(launch_pdl(kv_read_kernel<T, 64>, grid, dim3(kKvThreads), 0, s, kq, kscale, vq, vscale,
                                kt, ldk, vt, ldv, p));
    else
      DLM_CHECK_CUDA(launch_pdl(kv_read_kernel<T, 128>, grid, dim3(kKvThreads), 0, s, kq, kscale, vq, vscale,
                                kt, ldk, vt, ldv, p));
  });
  return DLM_OK;
}

}  // extern "C"
