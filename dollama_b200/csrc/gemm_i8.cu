// Matrix product in 8-bit integers with one scale per token and one per channel:
//
//   y[m, n] = T( float(sum_k xq[m, k] * wq[n, k]) * xscale[m] * wscale[n] (+ bias[n]) )
//
// on tcgen05.mma kind::i8.  The sum is exact (int32 accumulators in tensor memory, |sum| <= 128^2 K
// < 2^31); the epilogue is fp32 with one rounding to T.
//
// Two kernels, chosen by estimated time (launch_best):
//   gemm_i8_kernel     persistent, tiles of tokens x channels, double-buffered accumulators: a CTA
//                      pair (cta_group::2) per 256 x 256 tile, or a CTA per 128 x 128 tile.  Bound by
//                      the tensor cores and the power limit for large K (8192 x 8192 x 4096, fp16 out:
//                      177 us, 3100 TOP/s; with one CTA per 128 x 128 tile 329 us, bound by operand
//                      reads from L2, by their count: 128 bytes a clock and SM asked for).  Small K is
//                      far from both floors (4096 x 16000 x 512, fp16 out: 49 us, 22 by the bytes, 20
//                      by the operations; fp32 out 74 for 42): latencies of the epilogue, little of
//                      which four k-blocks hide (tensor pipe 34 %, issue slots 35 %, DRAM 19 %).  Odd
//                      N stores by elements: 1003 x 2111 x 1360 bf16 11.0 us, N = 2112 10.0;
//   gemm_i8_k_kernel   for few tokens: 128 channels (the MMA's M operand) x up to 128 tokens per
//                      cluster, whose CTAs split K and add their integer partial sums over
//                      distributed shared memory (integers: any order gives the same sum).  Bound by
//                      the weight's bytes and by latency (32 x 4096 x 4096: 6.5 us, the weight's bytes
//                      alone 2.6).
#include <cmath>
#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kBM = 128;  // rows of the MMA's M operand per CTA
constexpr int kKB = 128;  // k-block: 128 int8 = one 128-byte swizzled row
constexpr int kSubBytes = kBM * kKB;

struct GemmI8Params {
  const float* xs;
  const float* ws;
  const void* bias;
  void* y;
  long long ldy;
  int M, N, K;
  int m_tiles, n_tiles;
  int C;        // CTAs of a cluster (gemm_i8_k_kernel)
  int y_tma;    // y rows allow bulk-tensor stores
  int ws_vec;   // wscale allows 16-byte loads
  int* status;
};

// ================================================================== persistent kernel

constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + kEpiWarps * 32;
constexpr int kStageOut = 4096;  // an epilogue warp's staging: 32 rows of 128 bytes

// kPair: a pair of CTAs, each with its own 128 token rows and half of the 256 channels' weights in
// shared memory.  Two k-blocks per ring stage: the issuing thread's bookkeeping per stage costs about
// as much as one k-block's MMAs.
template <bool kPair>
struct Cfg {
  static constexpr int kBN = kPair ? 256 : 128;          // channels per tile
  static constexpr int kSub = 2;                         // k-blocks per stage
  static constexpr int kStageA = kSub * kSubBytes;       // this CTA's tokens
  static constexpr int kStageB = kSub * kSubBytes;       // this CTA's 128 channels
  static constexpr int kStages = 3;
  static constexpr int kSmem = kStages * (kStageA + kStageB) + kEpiWarps * kStageOut + 256 + 1024;
  static constexpr uint32_t kCols = 2 * kBN;
};
static_assert(Cfg<true>::kSmem <= 227 * 1024, "shared memory");

// Tile t in groups of 8 row tiles, rows fastest: the tiles of one wave share operands in L2.
__device__ __forceinline__ void tile_at(const GemmI8Params& p, int t, int& mt, int& nt) {
  constexpr int kGroup = 8;
  const int per = kGroup * p.n_tiles;
  const int g = t / per, r = t - g * per;
  const int rows = min(kGroup, p.m_tiles - g * kGroup);
  nt = r / rows;
  mt = g * kGroup + (r - nt * rows);
}

// wscale of 32 consecutive channels, the same for every lane; zero beyond N
__device__ __forceinline__ void channel_scales(const GemmI8Params& p, int n, float (&w)[32]) {
  if (p.ws_vec && n + 32 <= p.N) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p.ws + n) + j);
      w[4 * j] = f.x;
      w[4 * j + 1] = f.y;
      w[4 * j + 2] = f.z;
      w[4 * j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) w[j] = n + j < p.N ? __ldg(p.ws + n + j) : 0.0f;
  }
}

// This warp's 32 rows x `cols` channels of an accumulator (TMEM address ta) to y, 128 bytes of each
// row at a time through its staging buffer (16-byte pieces XORed with the row: no bank conflicts, and
// the layout that the 128-byte-swizzled tensor store reads).  A chunk is finished in registers before
// it waits for the buffer, so the previous chunk's store runs under it.
template <typename T>
__device__ __forceinline__ void epilogue(const GemmI8Params& p, const CUtensorMap* tmY, uint32_t ta, int row0,
                                         int n0, int cols, uint8_t* stage) {
  constexpr int kCols = 128 / static_cast<int>(sizeof(T));  // columns of a staged row
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 31;
  const float xs = row0 + lane < p.M ? p.xs[row0 + lane] : 0.0f;
  T* y = static_cast<T*>(p.y);
  const T* bias = static_cast<const T*>(p.bias);
  for (int c0 = 0; c0 < cols && n0 + c0 < p.N; c0 += kCols) {
    uint4 o[8];
#pragma unroll
    for (int h = 0; h < kCols; h += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(ta + c0 + h, r);
      float w[32];
      const int n = n0 + c0 + h;
      channel_scales(p, n, w);
      tmem_ld_wait();
      float v[32];
      if (bias) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = fmaf(static_cast<float>(static_cast<int>(r[j])) * xs, w[j], n + j < p.N ? to_f(bias[n + j]) : 0.0f);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = static_cast<float>(static_cast<int>(r[j])) * xs * w[j];
      }
#pragma unroll
      for (int q = 0; q < 32 / kPer; ++q) {
        Vec<T, kPer> t;
#pragma unroll
        for (int j = 0; j < kPer; ++j) t.v[j] = from_f<T>(v[q * kPer + j]);
        o[h / kPer + q] = *reinterpret_cast<const uint4*>(&t);
      }
    }
    if (p.y_tma) {  // the previous store has read the buffer
      if (lane == 0) bulk_wait_read_le0();
      __syncwarp();
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(stage + lane * 128 + ((q ^ (lane & 7)) << 4)) = o[q];
    // a bulk-tensor store writes whole 16-byte pieces: an odd last piece goes element by element
    if (p.y_tma && (n0 + c0 + kCols <= p.N || p.N % kPer == 0)) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (row0 < p.M) tma_store_2d(tmY, stage, n0 + c0, row0);
        bulk_commit_group();
      }
    } else {
      __syncwarp();
      const int rows = min(32, p.M - row0);
      for (int rr = 0; rr < rows; ++rr) {
        T* dst = y + static_cast<size_t>(row0 + rr) * p.ldy + n0 + c0;
#pragma unroll
        for (int h = 0; h < kCols; h += 32) {
          const int byte = (h + lane) * static_cast<int>(sizeof(T));
          if (n0 + c0 + h + lane < p.N)
            dst[h + lane] = *reinterpret_cast<const T*>(stage + rr * 128 + (((byte >> 4) ^ (rr & 7)) << 4) + (byte & 15));
        }
      }
      __syncwarp();
    }
  }
}

template <bool kPair, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_i8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmY, const GemmI8Params p) {
  using C = Cfg<kPair>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::kStages * C::kStageA;
  uint8_t* sOut = sB + C::kStages * C::kStageB;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + kEpiWarps * kStageOut);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;  // [2]
  uint64_t* tempty = tfull + 2;          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nkb = (p.K + kKB - 1) / kKB;
  const int tiles = p.m_tiles * p.n_tiles;
  const int rank = kPair ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = kPair ? blockIdx.x >> 1 : blockIdx.x, step = kPair ? gridDim.x >> 1 : gridDim.x;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (kPair ? 2 : 1) * kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc2(tmem_slot, C::kCols);
      tmem_relinquish2();
    } else {
      tmem_alloc(tmem_slot, C::kCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (kPair)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)

  if (warp == 0) {
    // ---- TMA: this CTA's 128 token rows and its 128 channels
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        int mt, nt;
        tile_at(p, t, mt, nt);
        const int a0 = (kPair ? 2 * mt + rank : mt) * kBM, b0 = (kPair ? 2 * nt + rank : nt) * 128;
        for (int kb = 0; kb < nkb; kb += C::kSub) {
          ok = mbar_wait(&empty[st], ph ^ 1, abort_flag, p.status, kDevTimeoutProducer);
          if (!ok) break;
          const int nsub = min(C::kSub, nkb - kb);
          // a pair's copies, both CTAs', complete on the even CTA's barrier
          if (!kPair || rank == 0) mbar_arrive_expect_tx(&full[st], (kPair ? 2 : 1) * nsub * 2 * kSubBytes);
          for (int u = 0; u < nsub; ++u) {
            uint8_t* da = sA + st * C::kStageA + u * kSubBytes;
            uint8_t* db = sB + st * C::kStageB + u * kSubBytes;
            if constexpr (kPair) {
              const uint32_t bar = pair_leader_addr(&full[st]);
              tma2_load_2d(da, &tmX, bar, (kb + u) * kKB, a0);
              tma2_load_2d(db, &tmW, bar, (kb + u) * kKB, b0);
            } else {
              tma_load_2d(da, &tmX, &full[st], (kb + u) * kKB, a0);
              tma_load_2d(db, &tmW, &full[st], (kb + u) * kKB, b0);
            }
          }
          if (++st == C::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA (the even CTA's thread issues for a pair)
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = idesc_s8_s32(kPair ? 256 : 128, C::kBN);
      const uint64_t da0 = sw128_desc(smem_u32(sA), 16, 1024);
      const uint32_t a_lo = static_cast<uint32_t>(da0), d_hi = static_cast<uint32_t>(da0 >> 32);
      const uint32_t b_lo = static_cast<uint32_t>(sw128_desc(smem_u32(sB), 16, 1024));
      int st = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step, ++i) {
        const int acc = i & 1;
        ok = mbar_wait(&tempty[acc], ((i >> 1) & 1) ^ 1, abort_flag, p.status, kDevTimeoutMma);
        tc_fence_after();
        const uint32_t d = tbase + static_cast<uint32_t>(acc * C::kBN);
        for (int kb = 0; kb < nkb && ok; kb += C::kSub) {
          ok = mbar_wait(&full[st], ph, abort_flag, p.status, kDevTimeoutMma);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            if (u > 0 && kb + u >= nkb) break;
            const uint32_t a = a_lo + static_cast<uint32_t>(st * C::kStageA + u * kSubBytes) / 16;
            const uint32_t b = b_lo + static_cast<uint32_t>(st * C::kStageB + u * kSubBytes) / 16;
#pragma unroll
            for (int k = 0; k < kKB / 32; ++k) {
              const uint32_t accumulate = (kb + u + k) != 0 ? 1u : 0u;
              if constexpr (kPair)
                umma2_i8_ss_lo(d, a + 2 * k, b + 2 * k, d_hi, idesc, accumulate);
              else
                umma_i8_ss(d, static_cast<uint64_t>(d_hi) << 32 | (a + 2 * k),
                           static_cast<uint64_t>(d_hi) << 32 | (b + 2 * k), idesc, accumulate);
            }
          }
          if constexpr (kPair)
            umma2_commit_mc(&empty[st], 0x3);
          else
            umma_commit(&empty[st]);
          if (++st == C::kStages) {
            st = 0;
            ph ^= 1;
          }
        }
        if (ok) {
          if constexpr (kPair)
            umma2_commit_mc(&tfull[acc], 0x3);
          else
            umma_commit(&tfull[acc]);
        }
      }
    }
    if (lane == 0) griddep_launch_dependents();
  } else {
    // ---- epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31, half of the channels
    const int quad = warp & 3, half = (warp - 2) >> 2;
    uint8_t* stage = sOut + (warp - 2) * kStageOut;
    int i = 0;
    for (int t = first; t < tiles; t += step, ++i) {
      int mt, nt;
      tile_at(p, t, mt, nt);
      const int acc = i & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (i >> 1) & 1, abort_flag, p.status, kDevTimeoutEpilogue)))
        break;
      tc_fence_after();
      const uint32_t ta = tbase + (static_cast<uint32_t>(quad * 32) << 16) +
                          static_cast<uint32_t>(acc * C::kBN + half * (C::kBN / 2));
      const int row0 = (kPair ? 2 * mt + rank : mt) * kBM + quad * 32;
      epilogue<T>(p, &tmY, ta, row0, nt * C::kBN + half * (C::kBN / 2), C::kBN / 2, stage);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair)
          mbar_arrive_cluster(&tempty[acc], 0);
        else
          mbar_arrive(&tempty[acc]);
      }
    }
    // the staging buffer must have been read before the CTA exits; the stores complete with the grid
    if (lane == 0) bulk_wait_read_le0();
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (kPair)
    cluster_sync_all();
  else
    __syncthreads();
  if (*abort_flag) drain_sleep(200000);
  if (warp == 1) {
    tc_fence_after();
    if constexpr (kPair)
      tmem_dealloc2(tbase, C::kCols);
    else
      tmem_dealloc(tbase, C::kCols);
  }
}

// ================================================================== split-K kernel

constexpr int kKThreads = 192;

template <int NT>
struct KCfg {
  static constexpr int kStageB = NT * kKB;
  static constexpr int kStages = NT <= 16 ? 6 : NT <= 32 ? 5 : 4;
  static constexpr int kRing = kStages * (kSubBytes + kStageB);
  static constexpr int kSmem = kRing + 256 + 1024;
  static constexpr uint32_t kCols = NT < 32 ? 32 : NT;
  static_assert(kRing >= kBM * NT * 4, "the partial sums reuse the ring");
};

__device__ __forceinline__ uint4 ld_dsmem16(uint32_t addr, uint32_t rank) {
  uint4 v;
  asm volatile(
      "{\n"
      ".reg .b32 ra;\n"
      "mapa.shared::cluster.u32 ra, %4, %5;\n"
      "ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [ra];\n"
      "}\n"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// A cluster of C CTAs: channels n0 .. n0 + 127 x tokens m0 .. m0 + NT - 1; CTA r multiplies its share
// of the k-blocks.
template <int NT, typename T>
__global__ void __launch_bounds__(kKThreads)
    gemm_i8_k_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                     const GemmI8Params p) {
  using C = KCfg<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::kStages * kSubBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kRing);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.C, tile = static_cast<int>(blockIdx.x) / p.C;
  const int n0 = (tile % p.n_tiles) * kBM, m0 = (tile / p.n_tiles) * NT;
  const int nkb = (p.K + kKB - 1) / kKB;
  const int kb0 = nkb * rank / p.C, kb1 = nkb * (rank + 1) / p.C;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
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
      int st = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[st], ph ^ 1, abort_flag, p.status, kDevTimeoutProducer)) break;
        mbar_arrive_expect_tx(&full[st], kSubBytes + C::kStageB);
        tma_load_2d(sA + st * kSubBytes, &tmW, &full[st], kb * kKB, n0);
        tma_load_2d(sB + st * C::kStageB, &tmX, &full[st], kb * kKB, m0);
        if (++st == C::kStages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_s8_s32(kBM, NT);
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait(&full[st], ph, abort_flag, p.status, kDevTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = smem_u32(sA + st * kSubBytes), b = smem_u32(sB + st * C::kStageB);
#pragma unroll
        for (int k = 0; k < kKB / 32; ++k)
          umma_i8_ss(tbase, sw128_desc(a + k * 32, 16, 1024), sw128_desc(b + k * 32, 16, 1024), idesc,
                     (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(&empty[st]);
        if (++st == C::kStages) {
          st = 0;
          ph ^= 1;
        }
      }
      if (ok) umma_commit(acc_full);
      griddep_launch_dependents();
    }
  } else {
    // partial sums [token][channel] into the ring, which the last MMA has left
    const int quad = warp & 3;
    if (__all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_flag, p.status, kDevTimeoutEpilogue))) {
      tc_fence_after();
      const uint32_t ta = tbase + (static_cast<uint32_t>(quad * 32) << 16);
      int* part = reinterpret_cast<int*>(smem) + quad * 32 + lane;
#pragma unroll
      for (int c = 0; c < NT; c += 16) {
        if (m0 + c >= p.M) break;
        uint32_t r[16];
        tmem_ld_32x32b_x16(ta + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kBM] = static_cast<int>(r[j]);
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (p.C > 1)
    cluster_sync_all();
  else
    __syncthreads();
  if (*abort_flag == 0) {
    // this CTA's share of the tile's tokens; a thread keeps four channels (their scales are read once,
    // read for every token they took three times the whole product at 128 tokens x 512)
    constexpr int kQuads = kBM / 4, kRowsPer = kKThreads / kQuads;
    const int rows = min(NT, p.M - m0);
    const int m1 = rows * (rank + 1) / p.C;
    const int qd = threadIdx.x % kQuads, n = n0 + 4 * qd;
    T* y = static_cast<T*>(p.y);
    const T* bias = static_cast<const T*>(p.bias);
    float w[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = n + j < p.N ? p.ws[n + j] : 0.0f;
      b[j] = bias && n + j < p.N ? to_f(bias[n + j]) : 0.0f;
    }
    if (n < p.N) {
#pragma unroll 4
      for (int m = rows * rank / p.C + threadIdx.x / kQuads; m < m1; m += kRowsPer) {
        const int q = m * kQuads + qd;
        const uint32_t addr = smem_u32(smem) + 16 * q;
        const float xs = p.xs[m0 + m];
        int s[4] = {0, 0, 0, 0};
        if (p.C == 1) {
          const uint4 v = reinterpret_cast<const uint4*>(smem)[q];
          s[0] = static_cast<int>(v.x);
          s[1] = static_cast<int>(v.y);
          s[2] = static_cast<int>(v.z);
          s[3] = static_cast<int>(v.w);
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < p.C) {
              const uint4 v = ld_dsmem16(addr, c);
              s[0] += static_cast<int>(v.x);
              s[1] += static_cast<int>(v.y);
              s[2] += static_cast<int>(v.z);
              s[3] += static_cast<int>(v.w);
            }
        }
        T* dst = y + static_cast<size_t>(m0 + m) * p.ldy + n;
        Vec<T, 4> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = from_f<T>(fmaf(static_cast<float>(s[j]) * xs, w[j], b[j]));
        if (p.y_tma && n + 4 <= p.N) {
          *reinterpret_cast<Vec<T, 4>*>(dst) = o;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.N) dst[j] = o.v[j];
        }
      }
    }
  }
  if (p.C > 1) cluster_sync_all();  // no CTA leaves while another reads its partial sums
  if (*abort_flag) drain_sleep(200000);
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, C::kCols);
  }
}

// ================================================================== launch

// [rows][K] int8 with a row stride of ld bytes, box [box_rows][128], 128-byte swizzle; elements
// beyond rows or K arrive as zeros.
bool tmap_i8(CUtensorMap* tm, const void* base, int rows, int K, long long ld, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(ld)};
  const uint32_t box[2] = {kKB, static_cast<uint32_t>(box_rows)};
  return encode_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T>
constexpr CUtensorMapDataType tmap_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

template <typename K, typename... Args>
cudaError_t launch_cluster(K kernel, int grid, int threads, int smem, int cluster, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool kPair, typename T>
int launch(const int8_t* xq, long long ldx, const int8_t* w, GemmI8Params p, cudaStream_t s) {
  using C = Cfg<kPair>;
  static bool done[64] = {false};
  DLM_CHECK_CUDA(allow_smem(gemm_i8_kernel<kPair, T>, C::kSmem, done));
  CUtensorMap tx, tw, ty{};
  if (!tmap_i8(&tx, xq, p.M, p.K, ldx, kBM) || !tmap_i8(&tw, w, p.N, p.K, p.K, 128)) return DLM_ERR_CUDA;
  if (p.y_tma) {
    const uint64_t dims[2] = {static_cast<uint64_t>(p.N), static_cast<uint64_t>(p.M)};
    const uint64_t strides[1] = {static_cast<uint64_t>(p.ldy) * sizeof(T)};
    const uint32_t box[2] = {128 / sizeof(T), 32};
    if (!encode_tmap(&ty, tmap_type<T>(), 2, p.y, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return DLM_ERR_CUDA;
  }
  const int bm = kPair ? 256 : 128;
  p.m_tiles = (p.M + bm - 1) / bm;
  p.n_tiles = (p.N + C::kBN - 1) / C::kBN;
  const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles;
  DLM_REQUIRE(tiles < (1ll << 30), DLM_ERR_UNSUPPORTED, "gemm_i8: too many tiles");
  const int slots = kPair ? num_sms() / 2 : num_sms();
  const int n = static_cast<int>(tiles < slots ? tiles : slots);
  if (kPair)
    DLM_CHECK_CUDA(launch_cluster(gemm_i8_kernel<kPair, T>, 2 * n, kThreads, C::kSmem, 2, s, tx, tw, ty, p));
  else
    DLM_CHECK_CUDA(launch_cluster(gemm_i8_kernel<kPair, T>, n, kThreads, C::kSmem, 1, s, tx, tw, ty, p));
  return DLM_OK;
}

// Clusters of C CTAs that run at once (they have to fit inside the groups of SMs that share a cluster,
// so this is less than the SMs divided by C).
template <int NT, typename T>
int resident_clusters(int C, int dev, int sms) {
  static int cache[64][4] = {{0}};
  const int i = C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3;
  if (dev >= 64) return sms / C;
  if (cache[dev][i] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(kKThreads);
    cfg.dynamicSmemBytes = KCfg<NT>::kSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = C;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, gemm_i8_k_kernel<NT, T>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = sms / C > 0 ? sms / C : 1;
    }
    cache[dev][i] = n;
  }
  return cache[dev][i];
}

// Estimated microseconds of a launch, fitted to measured times of 91 shapes (M 1..4096, N and K
// 512..16000): fixed part plus waves of tiles times their k-blocks.  Where two kernels are within a few
// percent either may be taken.
struct Estimate {
  double us;
  int C;  // of gemm_i8_k_kernel
};

double tiles_of(int M, int N, int bm, int bn) {
  return static_cast<double>((M + bm - 1) / bm) * ((N + bn - 1) / bn);
}

// 128 x 128 tiles, one per SM: 512 x 512 x 512 5.1 us, 1024 x 8192 x 4096 35.8 us
double estimate_single(int M, int N, int nkb, int sms) {
  return 3.6 + std::ceil(tiles_of(M, N, 128, 128) / sms) * (0.9 + 0.225 * nkb);
}
// 256 x 256 tiles, one per pair: 512 x 512 x 512 7.3 us, 1024 x 8192 x 4096 27.2 us
double estimate_pair(int M, int N, int nkb, int sms) {
  return 5.5 + std::ceil(tiles_of(M, N, 256, 256) / (sms / 2)) * (2.8 + 0.29 * nkb);
}
// K split over clusters; up to NT tokens: 32 x 4096 x 4096 6.7 us (128 x 128 tiles: 10.8 us)
template <int NT, typename T>
Estimate estimate_k(int M, int N, int nkb, int dev, int sms) {
  constexpr double kFixed = NT == 16 ? 3.4 : NT == 32 ? 4.4 : NT == 64 ? 5.9 : 8.0;
  constexpr double kBlock = NT == 16 ? 0.127 : NT == 32 ? 0.14 : NT == 64 ? 0.17 : 0.225;
  Estimate best{1e30, 1};
  for (int C = 1; C <= 8 && (C == 1 || nkb >= 2 * C); C *= 2) {
    const double waves = std::ceil(tiles_of(M, N, NT, 128) / resident_clusters<NT, T>(C, dev, sms));
    const double us = 2.0 + (C > 1 ? 0.3 : 0.0) + waves * (kFixed - 2.0 + ((nkb + C - 1) / C) * kBlock);
    if (us < best.us) best = Estimate{us, C};
  }
  return best;
}

template <int NT, typename T>
int launch_k(const int8_t* xq, long long ldx, const int8_t* w, GemmI8Params p, int C, cudaStream_t s) {
  using K = KCfg<NT>;
  CUtensorMap tx, tw;
  if (!tmap_i8(&tx, xq, p.M, p.K, ldx, NT) || !tmap_i8(&tw, w, p.N, p.K, p.K, kBM)) return DLM_ERR_CUDA;
  p.m_tiles = (p.M + NT - 1) / NT;
  p.n_tiles = (p.N + kBM - 1) / kBM;
  p.C = C;
  const long long ctas = static_cast<long long>(p.m_tiles) * p.n_tiles * C;
  DLM_REQUIRE(ctas < (1ll << 30), DLM_ERR_UNSUPPORTED, "gemm_i8: too many tiles");
  DLM_CHECK_CUDA(launch_cluster(gemm_i8_k_kernel<NT, T>, static_cast<int>(ctas), kKThreads, K::kSmem, C, s, tx, tw,
                                p));
  return DLM_OK;
}

// The kernel of least estimated time.
template <int NT, typename T>
int launch_best(const int8_t* xq, long long ldx, const int8_t* w, const GemmI8Params& p, cudaStream_t s) {
  static bool done[64] = {false};
  DLM_CHECK_CUDA(allow_smem(gemm_i8_k_kernel<NT, T>, KCfg<NT>::kSmem, done));
  const int nkb = (p.K + kKB - 1) / kKB;
  const int sms = num_sms();
  int dev = 0;
  DLM_CHECK_CUDA(cudaGetDevice(&dev));
  const double single = estimate_single(p.M, p.N, nkb, sms), pair = estimate_pair(p.M, p.N, nkb, sms);
  const Estimate split = estimate_k<NT, T>(p.M, p.N, nkb, dev, sms);
  if (split.us <= single && split.us <= pair) return launch_k<NT, T>(xq, ldx, w, p, split.C, s);
  if (pair < single) return launch<true, T>(xq, ldx, w, p, s);
  return launch<false, T>(xq, ldx, w, p, s);
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
  DLM_REQUIRE(reinterpret_cast<uintptr_t>(y) % e == 0 && reinterpret_cast<uintptr_t>(bias) % e == 0 &&
                  reinterpret_cast<uintptr_t>(xscale) % 4 == 0 && reinterpret_cast<uintptr_t>(wscale) % 4 == 0,
              DLM_ERR_INVALID, "gemm_i8: y, bias or a scale is not aligned to its element type");
  GemmI8Params p{xscale, wscale, bias, y, ldy, M, N, K, 0, 0, 1,
                 aligned16(y) && ldy % static_cast<int>(16 / e) == 0, aligned16(wscale), device_status_ptr()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    if (M <= 16) return launch_best<16, T>(xq, ldx, w, p, s);
    if (M <= 32) return launch_best<32, T>(xq, ldx, w, p, s);
    if (M <= 64) return launch_best<64, T>(xq, ldx, w, p, s);
    return launch_best<128, T>(xq, ldx, w, p, s);
  });
}
