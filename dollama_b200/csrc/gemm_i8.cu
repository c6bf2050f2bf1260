// Matrix product in 8-bit integers with one scale per token and one per channel:
//
//   y[m, n] = T( float(sum_k xq[m, k] * wq[n, k]) * xscale[m] * wscale[n] (+ bias[n]) )
//
// The sum is exact (int32 accumulators in tensor memory, |sum| <= 128^2 K < 2^31); the epilogue is
// fp32 with one rounding to T.
#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kBM = 128;    // rows of the MMA's M operand per tile
constexpr int kKB = 128;    // k-block: 128 int8 = one 128-byte swizzled row
constexpr int kThreads = 192;

template <int BN>
struct Cfg {
  static constexpr int kStageA = kBM * kKB, kStageB = BN * kKB;
  static constexpr int kStages = 6;
  static constexpr int kSmem = kStages * (kStageA + kStageB) + 512 + 1024;
  static constexpr uint32_t kCols = 2 * BN < 32 ? 32 : 2 * BN;
};

struct GemmI8Params {
  const float* xs;
  const float* ws;
  const void* bias;
  void* y;
  long long ldy;
  int M, N, K;
  int m_tiles, n_tiles;  // tiles of the MMA's M and N operands
  int vec;               // y rows allow 16-byte stores
  int* status;
};

// kSwap: the MMA's M operand is the weight (channels) and its N operand the tokens.
template <int BN, bool kSwap, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const GemmI8Params p) {
  using C = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::kStages * C::kStageA;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + C::kStages * C::kStageB);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;  // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = (p.K + kKB - 1) / kKB;
  const int tiles = p.m_tiles * p.n_tiles;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int a0 = (t % p.m_tiles) * kBM, b0 = (t / p.m_tiles) * BN;
        for (int kb = 0; kb < nkb; ++kb) {
          ok = mbar_wait(&empty[st], ph ^ 1, abort_flag, p.status, kDevTimeoutProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[st], C::kStageA + C::kStageB);
          tma_load_2d(sA + st * C::kStageA, &tmA, &full[st], kb * kKB, a0);
          tma_load_2d(sB + st * C::kStageB, &tmB, &full[st], kb * kKB, b0);
          if (++st == C::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_s8_s32(kBM, BN);
      int st = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x, ++i) {
        const int acc = i & 1;
        ok = mbar_wait(&tempty[acc], ((i >> 1) & 1) ^ 1, abort_flag, p.status, kDevTimeoutMma);
        tc_fence_after();
        const uint32_t d = tbase + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < nkb && ok; ++kb) {
          ok = mbar_wait(&full[st], ph, abort_flag, p.status, kDevTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = smem_u32(sA + st * C::kStageA), b = smem_u32(sB + st * C::kStageB);
#pragma unroll
          for (int k = 0; k < kKB / 32; ++k)
            umma_i8_ss(d, sw128_desc(a + k * 32, 16, 1024), sw128_desc(b + k * 32, 16, 1024), idesc,
                       (kb != 0 || k != 0) ? 1u : 0u);
          umma_commit(&empty[st]);
          if (++st == C::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
        if (ok) umma_commit(&tfull[acc]);
      }
      griddep_launch_dependents();
    }
  } else {
    // epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31
    const int quad = warp & 3;
    T* y = static_cast<T*>(p.y);
    const T* bias = static_cast<const T*>(p.bias);
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      const int acc = i & 1;
      const int a0 = (t % p.m_tiles) * kBM + quad * 32 + lane, b0 = (t / p.m_tiles) * BN;
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (i >> 1) & 1, abort_flag, p.status, kDevTimeoutEpilogue)))
        break;
      tc_fence_after();
      const uint32_t ta = tbase + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(acc * BN);
      const bool in = a0 < (kSwap ? p.N : p.M);
      const float sa = in ? (kSwap ? p.ws : p.xs)[a0] : 0.0f;
#pragma unroll 1
      for (int c = 0; c < BN; c += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(ta + c, r);
        tmem_ld_wait();
        if (kSwap) {
          const float bv = (in && bias) ? to_f(bias[a0]) : 0.0f;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int m = b0 + c + j;
            if (in && m < p.M)
              y[static_cast<size_t>(m) * p.ldy + a0] =
                  from_f<T>(fmaf(static_cast<float>(static_cast<int>(r[j])) * p.xs[m], sa, bv));
          }
        } else {
          Vec<T, 16 / sizeof(T)> o[sizeof(T)];
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int n = b0 + c + j;
            const float w = n < p.N ? p.ws[n] : 0.0f;
            const float bv = (bias && n < p.N) ? to_f(bias[n]) : 0.0f;
            v[j] = fmaf(static_cast<float>(static_cast<int>(r[j])) * sa, w, bv);
            o[j / (16 / sizeof(T))].v[j % (16 / sizeof(T))] = from_f<T>(v[j]);
          }
          if (in) {
            T* dst = y + static_cast<size_t>(a0) * p.ldy + b0 + c;
            if (p.vec && b0 + c + 16 <= p.N) {
#pragma unroll
              for (int q = 0; q < static_cast<int>(sizeof(T)); ++q)
                reinterpret_cast<Vec<T, 16 / sizeof(T)>*>(dst)[q] = o[q];
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (b0 + c + j < p.N) dst[j] = o[j / (16 / sizeof(T))].v[j % (16 / sizeof(T))];
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_sleep(200000);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, C::kCols);
  }
}

// [rows][K] int8 with a row stride of ld bytes, box [box_rows][128], 128-byte swizzle; elements
// beyond rows or K arrive as zeros.
bool tmap_i8(CUtensorMap* tm, const void* base, int rows, int K, long long ld, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {kKB, static_cast<uint32_t>(box_rows)};
  return encode_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int BN, bool kSwap, typename T>
int launch(const int8_t* xq, long long ldx, const int8_t* w, GemmI8Params p, cudaStream_t s) {
  static bool attr_set[64] = {false};
  int dev = 0;
  DLM_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !attr_set[dev]) {
    DLM_CHECK_CUDA(cudaFuncSetAttribute(gemm_i8_kernel<BN, kSwap, T>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::kSmem));
    if (dev < 64) attr_set[dev] = true;
  }
  CUtensorMap ta, tb;
  if (!tmap_i8(&ta, kSwap ? w : xq, kSwap ? p.N : p.M, p.K, kSwap ? p.K : ldx, kBM)) return DLM_ERR_CUDA;
  if (!tmap_i8(&tb, kSwap ? xq : w, kSwap ? p.M : p.N, p.K, kSwap ? ldx : p.K, BN)) return DLM_ERR_CUDA;
  p.m_tiles = ((kSwap ? p.N : p.M) + kBM - 1) / kBM;
  p.n_tiles = ((kSwap ? p.M : p.N) + BN - 1) / BN;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  DLM_REQUIRE(tiles < (1ll << 30), DLM_ERR_UNSUPPORTED, "gemm_i8: too many tiles");
  const int grid = static_cast<int>(tiles < num_sms() ? tiles : num_sms());
  DLM_CHECK_CUDA(launch_pdl(gemm_i8_kernel<BN, kSwap, T>, dim3(grid), dim3(kThreads), Cfg<BN>::kSmem, s, ta,
                            tb, p));
  return DLM_OK;
}

}  // namespace

}  // namespace dlm

extern "C" int dlm_gemm_i8(const int8_t* xq, int ldx, const float* xscale, const int8_t* w,
                           const float* wscale, const void* bias, void* y, int ldy, int M, int N, int K,
                           int dtype, void* stream) {
  using namespace dlm;
  DLM_REQUIRE(M >= 0 && N >= 0 && K >= 0, DLM_ERR_INVALID, "gemm_i8: negative size (M=%d, N=%d, K=%d)", M, N, K);
  DLM_REQUIRE(dtype_ok(dtype), DLM_ERR_INVALID, "gemm_i8: unknown dtype %d", dtype);
  if (M == 0 || N == 0 || K == 0) return DLM_OK;
  DLM_REQUIRE(xq && xscale && w && wscale && y, DLM_ERR_INVALID, "gemm_i8: null pointer");
  DLM_REQUIRE(K % 16 == 0 && ldx % 16 == 0 && ldx >= K, DLM_ERR_INVALID,
              "gemm_i8: K=%d and ldx=%d must be multiples of 16, ldx at least K", K, ldx);
  DLM_REQUIRE(K < (1 << 17), DLM_ERR_UNSUPPORTED, "gemm_i8: K=%d (the int32 sum holds K < 131072)", K);
  DLM_REQUIRE(ldy >= N, DLM_ERR_INVALID, "gemm_i8: ldy=%d is below N=%d", ldy, N);
  DLM_REQUIRE(aligned16(xq) && aligned16(w), DLM_ERR_INVALID, "gemm_i8: xq and w must be 16-byte aligned");
  const size_t e = dtype_size(dtype);
  DLM_REQUIRE(reinterpret_cast<uintptr_t>(y) % e == 0 && reinterpret_cast<uintptr_t>(bias) % e == 0,
              DLM_ERR_INVALID, "gemm_i8: y or bias is not aligned to its element type");
  GemmI8Params p{xscale, wscale, bias, y, ldy, M, N, K, 0, 0,
                 aligned16(y) && ldy % static_cast<int>(16 / e) == 0, device_status_ptr()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    if (M <= 16) return launch<16, true, T>(xq, ldx, w, p, s);
    if (M <= 64) return launch<64, true, T>(xq, ldx, w, p, s);
    return launch<128, false, T>(xq, ldx, w, p, s);
  });
}
