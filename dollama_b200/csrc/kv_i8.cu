// The int8 K/V cache of a language model: quantizing K and V rows as they are written, and reading
// them back.
//
// One row is the Dh values of one token and one head; its scale is a / 127 (a = largest magnitude)
// and its codes round_half_away(127 x / a), the rule of dlm_quantize_act_i8.  Codes are
// [B][H][Lmax][Dh], scales [B][H][Lmax], so a head's keys are contiguous for the attention that
// reads them.  Neighbouring lanes take the K row and the V row of one token and head.  Memory-bound:
// 16 sequences x 2048 tokens x 8 heads x 128, fp16, ragged: write 28.3 us (82 % of the measured copy
// rate), read 27.9 us (84 %) at best; both together 55 to 66 us from run to run.  The write takes 32 bytes of a row a lane: with 16, the bookkeeping of a
// row (its place in the cache, the divisions by a and 127) took 38.8 us; the read takes 8 values a lane:
// with 16, its 16-byte stores leave gaps between lanes (30.7 us).
#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kKvThreads = 256;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by Invariant Integers using
// Multiplication", 1994): q = (umulhi(n, mul) + n) >> shift with shift = ceil(log2 d), mul =
// floor(2^32 (2^shift - d) / d) + 1.
struct FastDiv {
  unsigned d, mul, shift;
  explicit FastDiv(unsigned v) : d(v), mul(0), shift(0) {
    while ((1ull << shift) < v) ++shift;
    mul = static_cast<unsigned>(((1ull << 32) * ((1ull << shift) - v)) / v + 1);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct KvShape {
  int B, S, H, Lmax;
  const int* pos;     // [B] position of each sequence's first new token
  const int* counts;  // [B] new tokens of each sequence, or null: S
  int* bad_position;  // device status word of positions
  unsigned units;     // B * S * H
  FastDiv by_h, by_s;
};

// values of a row that a lane takes
template <typename T>
constexpr int kWriteLane = 32 / static_cast<int>(sizeof(T));
constexpr int kReadLane = 8;

// kLane elements of a row in 16-byte pieces
template <typename T, int kLane>
struct Part {
  static constexpr int kPer = 16 / sizeof(T), kPieces = kLane / kPer;
  Vec<T, kPer> v[kPieces];
  __device__ __forceinline__ T& at(int i) { return v[i / kPer].v[i % kPer]; }
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) v[j] = reinterpret_cast<const Vec<T, kPer>*>(src)[j];
  }
  __device__ __forceinline__ void store(T* dst) const {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) reinterpret_cast<Vec<T, kPer>*>(dst)[j] = v[j];
  }
};

// Unit u is (token, head).  Whether its cache row exists: the token is below its sequence's count and
// its position inside the cache (a position outside raises the device status word of positions).
__device__ __forceinline__ bool locate(const KvShape& p, unsigned u, unsigned& tok, unsigned& hd, size_t& row) {
  if (u >= p.units) return false;
  tok = p.by_h.div(u);
  hd = u - tok * p.H;
  const unsigned b = p.by_s.div(tok);
  const int s = static_cast<int>(tok - b * p.S);
  if (s >= (p.counts ? p.counts[b] : p.S)) return false;
  const long long at = static_cast<long long>(p.pos[b]) + s;
  if (at < 0 || at >= p.Lmax) {
    if (p.bad_position) *p.bad_position = kDevBadPosition;
    return false;
  }
  row = (static_cast<size_t>(b) * p.H + hd) * p.Lmax + static_cast<size_t>(at);
  return true;
}

// Codes of this lane's values and their store; a: the row's largest magnitude (or NaN).
template <typename T, int kLane>
__device__ __forceinline__ void write_row(Part<T, kLane>& x, float a, int8_t* q, float* scale, bool first) {
  const bool finite = a < INFINITY;  // false for a NaN as well
  const double da = static_cast<double>(a);
  auto exact = [&](int j) { return quant_exact(static_cast<double>(to_f(x.at(j))), da); };
  uint32_t c[kLane / 4] = {};
  if (a >= 1e-30f && finite) {
    constexpr bool k16 = sizeof(T) == 2;
    const float rq = 127.0f / a * (k16 ? kHalvesAway : 1.0f);
    float v[kLane];
#pragma unroll
    for (int j = 0; j < kLane; ++j) v[j] = to_f(x.at(j)) * rq;
    if constexpr (k16)
      quant_codes_16<kLane>(v, c);
    else
      quant_codes<kLane>(v, 0x1p-15f, c, exact);  // two roundings: within 127 * 2^-23
  } else if (a > 0.0f && finite) {
    // 127 / a may leave fp32's range
#pragma unroll
    for (int j = 0; j < kLane; ++j) c[j / 4] |= (static_cast<uint32_t>(exact(j)) & 0xFFu) << (8 * (j % 4));
  }
  if constexpr (kLane == 16)
    *reinterpret_cast<uint4*>(q) = make_uint4(c[0], c[1], c[2], c[3]);
  else
    *reinterpret_cast<uint2*>(q) = make_uint2(c[0], c[1]);
  // a row that holds a NaN or an infinity: codes 0 under a NaN scale
  if (first) *scale = finite ? __fdiv_rn(a, 127.0f) : NAN;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kKvThreads)
    kv_append_kernel(const T* __restrict__ k, long long ldk, const T* __restrict__ v, long long ldv,
                     int8_t* __restrict__ kq, float* __restrict__ ks, int8_t* __restrict__ vq,
                     float* __restrict__ vs, const KvShape p) {
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  constexpr int kLane = kWriteLane<T>, G = DH / kLane;
  const unsigned u = blockIdx.x * (kKvThreads / G) + threadIdx.x / G;
  const int c = threadIdx.x % G;
  unsigned tok = 0, hd = 0;
  size_t row = 0;
  const bool live = locate(p, u, tok, hd, row);
  Part<T, kLane> xk, xv;
  float ak = 0.0f, av = 0.0f;
  if (live) {
    xk.load(k + tok * ldk + hd * DH + c * kLane);
    xv.load(v + tok * ldv + hd * DH + c * kLane);
#pragma unroll
    for (int j = 0; j < Part<T, kLane>::kPieces; ++j) {
      ak = max_abs(xk.v[j], ak);
      av = max_abs(xv.v[j], av);
    }
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    ak = max_nan(ak, __shfl_xor_sync(0xffffffffu, ak, o));
    av = max_nan(av, __shfl_xor_sync(0xffffffffu, av, o));
  }
  if (!live) return;
  write_row(xk, ak, kq + row * DH + c * kLane, ks + row, c == 0);
  write_row(xv, av, vq + row * DH + c * kLane, vs + row, c == 0);
}

template <typename T>
__device__ __forceinline__ Part<T, kReadLane> values(uint2 q, float scale) {
  Part<T, kReadLane> x;
#pragma unroll
  for (int j = 0; j < kReadLane; ++j) {
    const int code = static_cast<int>((j < 4 ? q.x : q.y) << (24 - 8 * (j % 4))) >> 24;
    x.at(j) = from_f<T>(static_cast<float>(code) * scale);
  }
  return x;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kKvThreads)
    kv_read_kernel(const int8_t* __restrict__ kq, const float* __restrict__ ks,
                   const int8_t* __restrict__ vq, const float* __restrict__ vs, T* __restrict__ k,
                   long long ldk, T* __restrict__ v, long long ldv, const KvShape p) {
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  constexpr int kLane = kReadLane, G = DH / kLane;
  const unsigned u = blockIdx.x * (kKvThreads / G) + threadIdx.x / G;
  const int c = threadIdx.x % G;
  unsigned tok, hd;
  size_t row;
  if (!locate(p, u, tok, hd, row)) return;
  const uint2 qk = *reinterpret_cast<const uint2*>(kq + row * DH + c * kLane);
  const uint2 qv = *reinterpret_cast<const uint2*>(vq + row * DH + c * kLane);
  const float sk = ks[row], sv = vs[row];
  values<T>(qk, sk).store(k + tok * ldk + hd * DH + c * kLane);
  values<T>(qv, sv).store(v + tok * ldv + hd * DH + c * kLane);
}

// The host checks of both calls; `empty` when there is nothing to do.
int check(const char* fn, const void* k, int ldk, const void* v, int ldv, const void* kq, const void* ks,
          const void* vq, const void* vs, int B, int S, int H, int Dh, int Lmax, const int* pos,
          const int* counts, int dtype, bool& empty) {
  empty = false;
  DLM_REQUIRE(B >= 0 && S >= 0 && H >= 0 && Lmax >= 0, DLM_ERR_INVALID, "%s: negative size", fn);
  DLM_REQUIRE(dtype_ok(dtype), DLM_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  DLM_REQUIRE(Dh == 64 || Dh == 128, DLM_ERR_UNSUPPORTED, "%s: head dim %d (64 or 128)", fn, Dh);
  empty = B == 0 || S == 0 || H == 0 || Lmax == 0;
  if (empty) return DLM_OK;
  DLM_REQUIRE(k && v && kq && ks && vq && vs && pos, DLM_ERR_INVALID, "%s: null pointer", fn);
  const long long width = static_cast<long long>(H) * Dh;
  DLM_REQUIRE(ldk >= width && ldv >= width, DLM_ERR_INVALID, "%s: a token stride is below H * Dh = %lld", fn,
              width);
  const int vec = static_cast<int>(16 / dtype_size(dtype));
  DLM_REQUIRE(aligned16(k) && aligned16(v) && ldk % vec == 0 && ldv % vec == 0, DLM_ERR_INVALID,
              "%s: k / v rows must start on 16-byte boundaries", fn);
  DLM_REQUIRE(aligned16(kq) && aligned16(vq), DLM_ERR_INVALID, "%s: cache codes must be 16-byte aligned", fn);
  DLM_REQUIRE(aligned4(ks) && aligned4(vs) && aligned4(pos) && aligned4(counts), DLM_ERR_INVALID,
              "%s: a scale or position array is not 4-byte aligned", fn);
  DLM_REQUIRE(static_cast<double>(B) * S * H < 2147483000.0, DLM_ERR_UNSUPPORTED, "%s: too many rows", fn);
  return DLM_OK;
}

KvShape shape(int B, int S, int H, int Lmax, const int* pos, const int* counts) {
  return KvShape{B, S, H, Lmax, pos, counts, device_position_ptr(), static_cast<unsigned>(B) * S * H,
                 FastDiv(H), FastDiv(S)};
}

dim3 grid_of(const KvShape& p, int Dh, int lane) {
  const unsigned per = kKvThreads / (Dh / lane);
  return dim3((p.units + per - 1) / per);
}

}  // namespace

}  // namespace dlm

extern "C" {

int dlm_kv_i8_append(const void* k, int ldk, const void* v, int ldv, int8_t* kq, float* kscale, int8_t* vq,
                     float* vscale, int B, int S, int H, int Dh, int Lmax, const int* pos,
                     const int* counts, int dtype, void* stream) {
  using namespace dlm;
  bool empty;
  const int rc = check("kv_i8_append", k, ldk, v, ldv, kq, kscale, vq, vscale, B, S, H, Dh, Lmax, pos, counts, dtype,
                       empty);
  if (rc != DLM_OK || empty) return rc;
  const KvShape p = shape(B, S, H, Lmax, pos, counts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    auto kernel = Dh == 64 ? kv_append_kernel<T, 64> : kv_append_kernel<T, 128>;
    DLM_CHECK_CUDA(launch_pdl(kernel, grid_of(p, Dh, kWriteLane<T>), dim3(kKvThreads), 0, s, static_cast<const T*>(k), ldk,
                              static_cast<const T*>(v), ldv, kq, kscale, vq, vscale, p));
  });
  return DLM_OK;
}

int dlm_kv_i8_read(const int8_t* kq, const float* kscale, const int8_t* vq, const float* vscale, void* k,
                   int ldk, void* v, int ldv, int B, int S, int H, int Dh, int Lmax, const int* pos,
                   const int* counts, int dtype, void* stream) {
  using namespace dlm;
  bool empty;
  const int rc = check("kv_i8_read", k, ldk, v, ldv, kq, kscale, vq, vscale, B, S, H, Dh, Lmax, pos, counts, dtype,
                       empty);
  if (rc != DLM_OK || empty) return rc;
  const KvShape p = shape(B, S, H, Lmax, pos, counts);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    auto kernel = Dh == 64 ? kv_read_kernel<T, 64> : kv_read_kernel<T, 128>;
    DLM_CHECK_CUDA(launch_pdl(kernel, grid_of(p, Dh, kReadLane), dim3(kKvThreads), 0, s, kq, kscale, vq, vscale,
                              static_cast<T*>(k), ldk, static_cast<T*>(v), ldv, p));
  });
  return DLM_OK;
}

}  // extern "C"
