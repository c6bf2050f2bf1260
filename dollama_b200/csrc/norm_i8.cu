// RMS norm with the residual's addition and an int8 output with one scale per token.
//
//   h[m, k] = T(x[m, k] + residual[m, k])          (stored when h_out is given)
//   p[m, k] = h[m, k] * w[k],  a_m = max_k |p[m, k]|
//   xscale[m] = a_m / (127 sqrt(mean_k h[m, k]^2 + eps))
//   xq[m, k] = round_half_away(127 p[m, k] / a_m)
//
// which is the quantization rule of dlm_quantize_act_i8 applied to h * w / rms: the factor 1 / rms
// is common to the row, so it leaves the codes and only scales xscale.  The codes are therefore
// those of the definition exactly: h is held in T, its product with w is exact in fp32 for 16-bit
// types (in double for fp32), and quotients next to a half-integer are formed in double.
//
// A row is read once, kept in registers, reduced once (sum of squares and largest magnitude
// together), and written once: 3 e + 1 bytes an element with a residual.  16384 x 4096 fp16: 84 us, 85 %
// of the measured copy rate (116 us when sums and products went through separate conversions: the
// instructions, not the bytes, were the bound).  Rows whose squares or
// products leave fp32's range (and all-zero rows) take a second pass over the registers in double.
#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kNormMaxK = 32768;

struct NormParams {
  const void* x;
  const void* r;
  const void* w;
  void* h;
  int8_t* q;
  float* scale;
  long long ldx, ldr, ldh;
  int M, K;
  float eps;
};

__device__ __forceinline__ double max_nan_d(double a, double b) { return (a > b || a != a) ? a : b; }

// One block of blockDim.x threads per row; thread t handles elements (i * blockDim.x + t) * VEC ..
// + VEC - 1 of step i.  NV > 0: at most NV steps, h in registers; NV == 0: any number, h in dynamic
// shared memory (each thread reads only what it wrote).
template <int NV>
constexpr int kNormMaxThreads = NV == 1 || NV == 2 ? 256 : 512;

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kNormMaxThreads<NV>) add_rms_norm_i8_kernel(const NormParams p) {
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  constexpr bool kWide = sizeof(T) == 4;  // products need double
  __shared__ float s_sum[32], s_max[32];
  __shared__ double s_dsum[32], s_dmax[32];
  const int nw = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  using V = Vec<T, VEC>;
  const T* __restrict__ w = static_cast<const T*>(p.w);
  const int row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.ldx;
  const T* r = p.r ? static_cast<const T*>(p.r) + static_cast<size_t>(row) * p.ldr : nullptr;
  T* ho = p.h ? static_cast<T*>(p.h) + static_cast<size_t>(row) * p.ldh : nullptr;
  extern __shared__ __align__(16) uint8_t s_row[];
  V h_reg[NV > 0 ? NV : 1];
  float p_reg[NV > 0 ? NV : 1][VEC];  // h * w in fp32
  const int steps = NV > 0 ? NV : (p.K + blockDim.x * VEC - 1) / (blockDim.x * VEC);
  auto H = [&](int i) -> V& {
    if constexpr (NV > 0)
      return h_reg[i];
    else
      return reinterpret_cast<V*>(s_row)[i * blockDim.x + threadIdx.x];
  };
  float ss = 0.0f, amax = 0.0f;
  double damax = 0.0;
  V r_reg[NV > 0 ? NV : 1];
#pragma unroll(NV > 0 ? NV : 1)
  for (int i = 0; i < steps; ++i) {
    const int k = (i * blockDim.x + threadIdx.x) * VEC;
    if (k < p.K) {
      H(i) = *reinterpret_cast<const V*>(x + k);
      if constexpr (NV > 0)
        if (r) r_reg[i] = *reinterpret_cast<const V*>(r + k);
    }
  }
#pragma unroll(NV > 0 ? NV : 1)
  for (int i = 0; i < steps; ++i) {
    const int k = (i * blockDim.x + threadIdx.x) * VEC;
    if (k >= p.K) continue;
    V hv = H(i);
    if (r) {
      add_to(hv, NV > 0 ? r_reg[NV > 0 ? i : 0] : *reinterpret_cast<const V*>(r + k));
      H(i) = hv;
    }
    if (ho) *reinterpret_cast<V*>(ho + k) = hv;
    const V wv = *reinterpret_cast<const V*>(w + k);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      ss = fma_f(hv.v[j], hv.v[j], ss);
      const float f = fma_f(hv.v[j], wv.v[j], 0.0f);
      if constexpr (NV > 0) p_reg[i][j] = f;
      if constexpr (kWide)
        damax = max_nan_d(fabs(static_cast<double>(to_f(hv.v[j])) * static_cast<double>(to_f(wv.v[j]))), damax);
      else
        amax = max_nan(amax, fabsf(f));
    }
  }
  if constexpr (kWide) amax = static_cast<float>(damax);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (kWide)
      damax = max_nan_d(__shfl_xor_sync(0xffffffffu, damax, o), damax);
    else
      amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  if (nw > 1) {
    if (lane == 0) {
      s_sum[warp] = ss;
      s_max[warp] = amax;
      s_dmax[warp] = damax;
    }
    __syncthreads();
    ss = 0.0f;
    for (int i = 0; i < nw; ++i) {
      ss += s_sum[i];
      if constexpr (kWide)
        damax = max_nan_d(s_dmax[i], damax);
      else
        amax = max_nan(amax, s_max[i]);
    }
  }
  if constexpr (kWide)
    amax = static_cast<float>(damax);
  else
    damax = static_cast<double>(amax);
  // sums and products well inside fp32's range: their relative errors are fp32's
  const bool plain = ss > 1e-25f && ss < 1e30f && amax > 1e-25f && amax < 1e30f;
  double dscale = 0.0;
  if (!plain) {  // the same for every thread of the row
    double dss = 0.0;
    damax = 0.0;
#pragma unroll(NV > 0 ? NV : 1)
    for (int i = 0; i < steps; ++i) {
      const int k = (i * blockDim.x + threadIdx.x) * VEC;
      if (k >= p.K) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const double f = static_cast<double>(to_f(H(i).v[j]));
        dss = fma(f, f, dss);
        damax = max_nan_d(fabs(f * static_cast<double>(to_f(w[k + j]))), damax);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      dss += __shfl_xor_sync(0xffffffffu, dss, o);
      damax = max_nan_d(__shfl_xor_sync(0xffffffffu, damax, o), damax);
    }
    if (nw > 1) {
      __syncthreads();  // s_dmax of the first reduction has been read
      if (lane == 0) {
        s_dsum[warp] = dss;
        s_dmax[warp] = damax;
      }
      __syncthreads();
      dss = 0.0;
      for (int i = 0; i < nw; ++i) {
        dss += s_dsum[i];
        damax = max_nan_d(s_dmax[i], damax);
      }
    }
    dscale = damax / (127.0 * sqrt(dss / p.K + static_cast<double>(p.eps)));
    // a NaN or an infinity in the row (or its weights): codes 0 under a NaN scale, so that what is
    // computed from the row is NaN too
    if (!(dss < INFINITY && damax < INFINITY)) dscale = NAN;
    if (damax == 0.0) dscale = dss < INFINITY ? 0.0 : NAN;
  }
  if (threadIdx.x == 0)
    p.scale[row] = plain ? amax / (127.0f * sqrtf(ss / static_cast<float>(p.K) + p.eps))
                         : static_cast<float>(dscale);
  const float rq = 127.0f / amax;
  int8_t* qo = p.q + static_cast<size_t>(row) * p.K;
  // 127 / a and its product: within 127 * 2^-23 for exact products and a, twice that otherwise
  constexpr float kErr = kWide ? 0x1p-14f : 0x1p-15f;
  // codes of N values at a time: of one vector, or (VEC == 1) of four steps
  constexpr int N = VEC == 1 ? 4 : VEC, kStep = VEC == 1 ? 4 : 1;
#pragma unroll(NV > 0 ? NV : 1)
  for (int i = 0; i < steps; i += kStep) {
    // value j of the N: its step, its place in the row
    auto step = [&](int j) { return VEC == 1 ? i + j : i; };
    auto at = [&](int j) {
      return VEC == 1 ? (i + j) * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)
                      : (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * VEC + j;
    };
    if (at(0) >= p.K) continue;
    auto exact = [&](int j) {
      const T hj = H(step(j)).v[VEC == 1 ? 0 : j];
      return quant_exact(static_cast<double>(to_f(hj)) * static_cast<double>(to_f(w[at(j)])), damax);
    };
    float v[N];
    uint32_t c[N / 4];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bool in = VEC > 1 || at(j) < p.K;
      if constexpr (NV > 0)
        v[j] = in ? p_reg[step(j)][VEC == 1 ? 0 : j] * rq : 0.0f;
      else
        v[j] = in ? fma_f(H(step(j)).v[VEC == 1 ? 0 : j], w[at(j)], 0.0f) * rq : 0.0f;
    }
    if (plain) {
      quant_codes<N>(v, kErr, c, exact);
    } else {
      const bool some = damax > 0.0 && dscale == dscale;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool in = some && (VEC > 1 || at(j) < p.K);
        const uint32_t code = in ? static_cast<uint32_t>(exact(j)) & 0xFFu : 0u;
        c[j / 4] = (j % 4 ? c[j / 4] : 0u) | code << (8 * (j % 4));
      }
    }
    if constexpr (VEC == 1) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at(j) < p.K) qo[at(j)] = static_cast<int8_t>(c[0] >> (8 * j) & 0xFFu);
    } else if constexpr (VEC == 4) {
      *reinterpret_cast<uint32_t*>(qo + at(0)) = c[0];
    } else {
      *reinterpret_cast<uint2*>(qo + at(0)) = make_uint2(c[0], c[1]);
    }
  }
}

template <typename T, int VEC>
int launch_norm(const NormParams& p, cudaStream_t s) {
  const int n = p.K / VEC;  // vectors of a row
  auto go = [&](auto kernel, int nv) {
    const int threads = ((n + nv - 1) / nv + 31) / 32 * 32;
    return launch_pdl(kernel, dim3(p.M), dim3(threads), 0, s, p);
  };
  if (VEC == 1 && n <= 4096) {
    DLM_CHECK_CUDA(go(add_rms_norm_i8_kernel<T, VEC, (VEC == 1 ? 8 : 0)>, 8));
  } else if (VEC > 1 && n <= 256) {
    DLM_CHECK_CUDA(go(add_rms_norm_i8_kernel<T, VEC, (VEC > 1 ? 1 : 0)>, 1));
  } else if (VEC > 1 && n <= 512) {
    DLM_CHECK_CUDA(go(add_rms_norm_i8_kernel<T, VEC, (VEC > 1 ? 2 : 0)>, 2));
  } else if (VEC > 1 && n <= 2048) {
    DLM_CHECK_CUDA(go(add_rms_norm_i8_kernel<T, VEC, (VEC > 1 ? 4 : 0)>, 4));
  } else {
    const int threads = n >= 2048 ? 512 : n >= 512 ? 256 : (n + 31) / 32 * 32;
    const size_t smem = static_cast<size_t>((n + threads - 1) / threads) * threads * VEC * sizeof(T);
    auto kernel = add_rms_norm_i8_kernel<T, VEC, 0>;
    // always: the static arrays share the 48 KB that a kernel has without leave, so a row of just that
    // size needs it too
    static bool done[64] = {false};
    DLM_CHECK_CUDA(allow_smem(kernel, static_cast<int>((kNormMaxK + 512) * sizeof(T)), done));
    DLM_CHECK_CUDA(launch_pdl(kernel, dim3(p.M), dim3(threads), smem, s, p));
  }
  return DLM_OK;
}

}  // namespace

}  // namespace dlm

extern "C" int dlm_add_rms_norm_i8(const void* x, int ldx, const void* residual, int ldr,
                                   const void* weight, void* h_out, int ldh, int8_t* xq, float* xscale,
                                   int M, int K, float eps, int dtype, void* stream) {
  using namespace dlm;
  DLM_REQUIRE(M >= 0 && K >= 0, DLM_ERR_INVALID, "add_rms_norm_i8: negative size (M=%d, K=%d)", M, K);
  DLM_REQUIRE(dtype_ok(dtype), DLM_ERR_INVALID, "add_rms_norm_i8: unknown dtype %d", dtype);
  if (M == 0 || K == 0) return DLM_OK;
  DLM_REQUIRE(x && weight && xq && xscale, DLM_ERR_INVALID, "add_rms_norm_i8: null pointer");
  DLM_REQUIRE(K <= kNormMaxK, DLM_ERR_UNSUPPORTED, "add_rms_norm_i8: K=%d (at most %d)", K,
              kNormMaxK);
  DLM_REQUIRE(ldx >= K && (!residual || ldr >= K) && (!h_out || ldh >= K), DLM_ERR_INVALID,
              "add_rms_norm_i8: a row stride is below K=%d", K);
  DLM_REQUIRE(eps > 0.0f && eps < INFINITY, DLM_ERR_INVALID, "add_rms_norm_i8: eps must be positive");
  const size_t e = dtype_size(dtype);
  auto al = [&](const void* q, size_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) == 0; };
  DLM_REQUIRE(al(x, e) && al(residual, e) && al(weight, e) && al(h_out, e) && al(xscale, 4),
              DLM_ERR_INVALID, "add_rms_norm_i8: a pointer is not aligned to its element type");
  NormParams p{x, residual, weight, h_out, xq, xscale, ldx, ldr, ldh, M, K, eps};
  // 16-byte accesses where every row of every operand starts on their boundary
  const int v = static_cast<int>(16 / e);
  auto row16 = [&](const void* q, long long ld) { return !q || (aligned16(q) && ld % v == 0); };
  const bool wide = K % v == 0 && row16(x, ldx) && row16(residual, ldr) && row16(h_out, ldh) &&
                    aligned16(weight) && al(xq, v);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    if (wide) return launch_norm<T, 16 / sizeof(T)>(p, s);
    return launch_norm<T, 1>(p, s);
  });
}
