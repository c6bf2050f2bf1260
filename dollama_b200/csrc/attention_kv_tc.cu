// Attention over the int8 K/V cache for many rows (prompt chunks), on tcgen05 (attention_kv.cu has
// the formulas and the few-row kernel).
//
// One CTA takes 128 rows of one (sequence, kv head): row r is TMEM lane r.  Its tiles of 64 keys
// alternate between two streams A and B, each with two score buffers and its own output accumulator,
// so that a stream's next scores are there when the softmax comes to them, and one stream's
// latencies lie under the other's softmax; a cluster of C CTAs may share a tile's keys.  All partial
// results meet at the end in a fixed order (A with B in the CTA, then the CTAs).
//   warps 0..3 / 4..7   softmax of stream A / B: S from TMEM, weights w = p vscale against each row's
//                       running reference, as fp16 pairs back into S's columns, from where the second
//                       product takes its A operand.  A lane takes two of eight columns of four rows
//                       (the 16x256b pieces), so that a key's scales, read from shared memory, serve
//                       four scores;
//   warps 8 / 9         MMA issuers of A / B: S = Q K^T (M 128, N 64, K DH), O += W V (M 128, N DH,
//                       K 64, V as an MN-major operand); a buffer's next S follows its W V;
//   the other warps     the tiles' codes -> fp16 in the 128-byte-swizzled layout both products read,
//                       with the tile's scales, through a ring of kStages tiles (the next tile's
//                       codes are requested before the current one is converted).
// The scales stay outside the products, as in the few-row kernel: codes are exact in fp16, and so is q,
// each row scaled by a power of two for bf16 and fp32 (a row's result does not depend on its
// neighbours).  For fp32 inputs q and the weights are two fp16 terms each, and every product is issued
// for both.  Bound by the softmax and its hand-overs: 2 x 500 queries of 16 heads on 4 over 4096 keys,
// bf16, 44 us, of which 29 us remain when the softmax does nothing but pass its tiles on; the
// exponentials alone take 10.  512 threads of 128 registers leave the softmax warps 20 to 76 bytes of
// spills (by type and head dim).
#include "attention_kv.cuh"

namespace dlm {

namespace {

constexpr int kRows = 128;
constexpr int kTcThreads = 512;  // 4 warpgroups: softmax A, softmax B, MMA issuers, conversion
constexpr int kConvThreads = 128;

constexpr int KT = 64;  // keys per tile

// A cluster's CTAs wait for one another and for their tensor memory, all 512 columns.  Beside another
// stream's clusters that hold some (dlm_gemm_i8's split-K kernel would fit next to the 119 KB of Dh 64)
// each could hold the columns that the other's peer waits for, without end: so a CTA of a cluster takes
// an SM's whole shared memory, and has the columns as soon as it runs.
constexpr int kWholeSm = 227 * 1024;

template <int DH, bool kSplit>
struct TcCfg {
  static constexpr int NT = kSplit ? 2 : 1;  // fp16 terms of q and of the weights
  static constexpr int kHalves = DH / 64;    // 64-channel blocks (128-byte rows)
  static constexpr int kQBytes = NT * kHalves * kRows * 128;
  static constexpr int kTile = kHalves * KT * 128;  // K or V of a tile
  static constexpr int kStages = DH == 64 ? 6 : 4;
  static constexpr int kScales = 2 * KT * 4;  // kscale, vscale
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kOut = kRows * DH * 4;  // O of stream B, then the CTA's, over Q and the ring
  static constexpr int kData = kQBytes + kRing > kOut ? kQBytes + kRing : kOut;
  static constexpr int kSmem = kData + kStages * kScales + kRows * 5 * 4 + 512 + 1024;
  // TMEM columns: two S buffers of each stream (the weights' terms replace the scores, KT / 2 columns
  // each), then the streams' O
  static constexpr uint32_t kO = 4 * KT;
  static_assert(kO + 2 * DH <= 512 && NT * KT / 2 <= KT, "tensor memory");
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// Weights from here on do not say how far their reference is too low (they may have overflowed).
constexpr float kFarWeight = 1e30f;

// 16 codes -> 16 fp16 values (two 16-byte pieces)
__device__ __forceinline__ void expand16(uint4 c, uint4& a, uint4& b) {
  const uint32_t x = c.x ^ 0x80808080u, y = c.y ^ 0x80808080u, z = c.z ^ 0x80808080u, w = c.w ^ 0x80808080u;
  a = make_uint4(code_pair(x, 0x4140), code_pair(x, 0x4342), code_pair(y, 0x4140), code_pair(y, 0x4342));
  b = make_uint4(code_pair(z, 0x4140), code_pair(z, 0x4342), code_pair(w, 0x4140), code_pair(w, 0x4342));
}

template <typename T, int DH>
__global__ void __launch_bounds__(kTcThreads, 1)
    attn_kv_tc_kernel(const AttnKvParams p) {
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr bool kScaled = !std::is_same<T, __half>::value;
  using C = TcCfg<DH, kSplit>;
  constexpr int NT = C::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + C::kQBytes;
  float* sScale = reinterpret_cast<float*>(smem + C::kData);  // [stage][2][KT]
  float* s_ref = sScale + C::kStages * 2 * KT;                // [2][kRows] of A and B, then of the CTA
  float* s_l = s_ref + 2 * kRows;                             // [2][kRows]
  float* s_qmul = s_l + 2 * kRows;                            // [kRows] takes a row's scaling back
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_qmul + kRows);
  uint64_t* kv_full = bars;                  // [stages]
  uint64_t* kv_empty = kv_full + C::kStages; // [stages]
  uint64_t* s_full = kv_empty + C::kStages;  // [stream][buffer]
  uint64_t* w_full = s_full + 4;             // [stream][buffer]
  uint64_t* o_full = w_full + 4;             // [stream]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x % p.C);
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&kv_full[s], kConvThreads);
      mbar_init(&kv_empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&w_full[s], kRows);
    }
    for (int s = 0; s < 2; ++s) mbar_init(&o_full[s], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  const AttnKvTile tile(p, static_cast<int>(blockIdx.x / p.C), kRows, threadIdx.x == 0);
  const int n_tiles = (tile.n_keys + KT - 1) / KT;
  // this CTA's tiles: rank + C * i, i = 0, 1, ..; tile i belongs to stream i & 1, stage i % kStages
  const int n_mine = n_tiles > rank ? (n_tiles - rank + p.C - 1) / p.C : 0;

  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  if (warp < 4) {
    // ---- q as fp16 terms in shared memory (thread = row), rows beyond the last as zeros
    const int row = threadIdx.x;
    const bool q_in = tile.r0 + row <= tile.last;
    const T* q = tile.q_row<T>(p, q_in ? tile.r0 + row : 0, DH);
    float up = 1.0f;
    if constexpr (kScaled) {
      float mx = 0.0f;
      if (q_in)
        for (int i = 0; i < DH / kPer; ++i) {
          const Vec<T, kPer> v = reinterpret_cast<const Vec<T, kPer>*>(q)[i];
#pragma unroll
          for (int j = 0; j < kPer; ++j) mx = fmaxf(mx, fabsf(to_f(v.v[j])));
        }
      const int e = q_up(mx);
      up = pow2i(e);
      s_qmul[row] = p.scale_log2 * pow2i(-e);
    }
#pragma unroll
    for (int i = 0; i < DH / 8; ++i) {
      float f[8];
#pragma unroll
      for (int h = 0; h < 8 / kPer; ++h) {
        Vec<T, kPer> v;
        if (q_in) v = reinterpret_cast<const Vec<T, kPer>*>(q)[i * (8 / kPer) + h];
#pragma unroll
        for (int j = 0; j < kPer; ++j) f[h * kPer + j] = q_in ? to_f(v.v[j]) * up : 0.0f;
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hi[j] = half_pair(f[2 * j], f[2 * j + 1]);
        lo[j] = kSplit ? half_rest(hi[j], f[2 * j], f[2 * j + 1]) : 0u;
      }
      uint8_t* dst = sQ + (i / 8) * kRows * 128 + row * 128 + (((i % 8) ^ (row & 7)) << 4);
      *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (kSplit)
        *reinterpret_cast<uint4*>(dst + C::kHalves * kRows * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;

  if (warp >= 12) {
    // ================================================================ codes -> fp16
    const int t = threadIdx.x - 384;
    constexpr int kPieces = DH / 16;                    // 16-code pieces of a row
    constexpr int kEach = KT * kPieces / kConvThreads;  // pieces a thread converts, of K and of V
    const size_t head = tile.head(p);
    const int8_t* kb = p.kq + head * p.Lmax * DH;
    const int8_t* vb = p.vq + head * p.Lmax * DH;
    const float* ksb = p.ks + head * p.Lmax;
    const float* vsb = p.vs + head * p.Lmax;
    uint4 rk[kEach], rv[kEach];
    float sk = 0.0f, sv = 0.0f;
    auto request = [&](int i) {
      const int k0 = (rank + p.C * i) * KT;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int id = e * kConvThreads + t;
        const bool in = k0 + id / kPieces < tile.n_keys;
        const size_t off = static_cast<size_t>(k0) * DH + static_cast<size_t>(id) * 16;
        rk[e] = in ? __ldg(reinterpret_cast<const uint4*>(kb + off)) : make_uint4(0, 0, 0, 0);
        rv[e] = in ? __ldg(reinterpret_cast<const uint4*>(vb + off)) : make_uint4(0, 0, 0, 0);
      }
      const bool in = t < KT && k0 + t < tile.n_keys;
      sk = in ? __ldg(ksb + k0 + t) : 0.0f;
      sv = in ? __ldg(vsb + k0 + t) : 0.0f;
    };
    if (n_mine > 0) request(0);
    int st = 0;
    uint32_t ph = 0;
    for (int i = 0; i < n_mine; ++i) {
      if (!mbar_wait(&kv_empty[st], ph ^ 1, abort_flag, p.status, kDevTimeoutProducer)) break;
      uint8_t* dk = sKV + st * 2 * C::kTile;
      uint8_t* dv = dk + C::kTile;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int id = e * kConvThreads + t;
        const int r = id / kPieces, ch = id % kPieces;
        // the second half's pieces go in the other order: no bank conflict with the first half's
        const int odd = DH == 128 ? ch >> 2 : 0;
        const int off = (ch >> 2) * KT * 128 + r * 128;
        const int p0 = ((2 * (ch & 3) + odd) ^ (r & 7)) << 4, p1 = ((2 * (ch & 3) + 1 - odd) ^ (r & 7)) << 4;
        uint4 a, b;
        expand16(rk[e], a, b);
        *reinterpret_cast<uint4*>(dk + off + p0) = odd ? b : a;
        *reinterpret_cast<uint4*>(dk + off + p1) = odd ? a : b;
        expand16(rv[e], a, b);
        *reinterpret_cast<uint4*>(dv + off + p0) = odd ? b : a;
        *reinterpret_cast<uint4*>(dv + off + p1) = odd ? a : b;
      }
      if (t < KT) {
        sScale[st * 2 * KT + t] = kScaled ? sk : sk * p.scale_log2;
        sScale[st * 2 * KT + KT + t] = sv;
      }
      if (i + 1 < n_mine) request(i + 1);
      fence_proxy_async_smem();
      mbar_arrive(&kv_full[st]);
      if (++st == C::kStages) {
        st = 0;
        ph ^= 1;
      }
    }
  } else if (warp >= 8) {
    // ================================================================ MMA issuer of one stream
    const int sm = __shfl_sync(0xffffffffu, warp, 0) - 8;
    if (sm < 2) {
      constexpr uint32_t idesc_s = idesc_f16_f32(kRows, KT, false);
      constexpr uint32_t idesc_o = idesc_f16_f32(kRows, DH, true);
      const uint32_t to = tbase + C::kO + sm * DH;
      const int n_own = (n_mine - sm + 1) / 2;  // tiles of this stream
      auto wait = [&](uint64_t* bar, int parity) {
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.status, kDevTimeoutMma));
        tc_fence_after();
        return ok;
      };
      const uint64_t q_desc = sw128_desc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sw128_desc(smem_u32(sKV), 16, 1024);
      const uint64_t v_desc = sw128_desc(smem_u32(sKV) + C::kTile, KT * 128, 1024);
      int k_st = sm;                         // stage of the next scores' tile
      uint32_t k_ph = 0;
      auto step = [](int& st, uint32_t& ph) {  // the stream's next tile: two stages on
        st += 2;
        if (st >= C::kStages) {
          st -= C::kStages;
          ph ^= 1;
        }
      };
      // S of the stream's tile n (the CTA's tile 2 n + sm), once its codes are there
      auto scores = [&](int n) -> bool {
        if (!wait(&kv_full[k_st], k_ph)) return false;
        const uint64_t kd = k_desc + static_cast<uint32_t>(k_st * 2 * C::kTile) / 16;
        const uint32_t ts = tbase + (2 * sm + (n & 1)) * KT;
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int h = 0; h < C::kHalves; ++h)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_f16_ss(ts, q_desc + ((x * C::kHalves + h) * kRows * 128 + k * 32) / 16,
                            kd + (h * KT * 128 + k * 32) / 16, idesc_s, (x | h | k) != 0 ? 1u : 0u);
          umma_commit(&s_full[2 * sm + (n & 1)]);
        }
        __syncwarp();
        step(k_st, k_ph);
        return true;
      };
      bool ok = (n_own < 1 || scores(0)) && (n_own < 2 || scores(1));
      int st = sm;
      uint32_t ph = 0;
      for (int n = 0; ok && n < n_own; ++n) {
        const int buf = 2 * sm + (n & 1);
        ok = wait(&w_full[buf], (n >> 1) & 1);
        if (!ok) break;
        const uint64_t vd = v_desc + static_cast<uint32_t>(st * 2 * C::kTile) / 16;
        const uint32_t tw = tbase + buf * KT;
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
              umma_f16_ts(to, tw + x * (KT / 2) + k * 8, vd + k * 2048 / 16, idesc_o, (n | x | k) != 0 ? 1u : 0u);
          umma_commit(&kv_empty[st]);
          umma_commit(&o_full[sm]);
        }
        __syncwarp();
        step(st, ph);
        // the buffer's next scores replace the weights that this product reads
        if (n + 2 < n_own) ok = wait(&o_full[sm], n & 1) && scores(n + 2);
      }
      griddep_launch_dependents();
    }
  } else {
    // ================================================================ softmax of one stream
    const int sm = warp >> 2, gr = lane >> 2, c4 = lane & 3;
    const int row0 = (warp & 3) * 32 + gr;  // this lane's rows: row0 + 8 y
    constexpr uint32_t kHalf = 16u << 16;   // TMEM address of 16 lanes further
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t to = tbase + lanes + C::kO + sm * DH;
    float ref[4], l[4], qmul[4];
    int lim[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int r = tile.r0 + row0 + 8 * y;
      ref[y] = kNoRef;
      l[y] = 0.0f;
      qmul[y] = kScaled ? s_qmul[row0 + 8 * y] : 1.0f;
      lim[y] = r <= tile.last ? tile.seen(p, r) : tile.n_keys;
    }
    int n = 0;
    bool ok = true;
    for (int i = sm; i < n_mine && ok; i += 2, ++n) {
      const float* sc = sScale + (i % C::kStages) * 2 * KT + 2 * c4;
      const int k0 = (rank + p.C * i) * KT + 2 * c4;
      const bool masked = (rank + p.C * i) * KT + KT > tile.n_all;
      const int buf = 2 * sm + (n & 1);
      const uint32_t ts = tbase + lanes + buf * KT;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_full[buf], (n >> 1) & 1, abort_flag, p.status, kDevTimeoutSoftmax));
      if (!ok) break;
      tc_fence_after();
      // columns 32 q .. + 31 of this warp's rows: s[lane half]
      auto load = [&](int q, uint32_t (&s)[2][16]) {
        tmem_ld_16x256b_x4(ts + 32 * q, s[0]);
        tmem_ld_16x256b_x4(ts + kHalf + 32 * q, s[1]);
        tmem_ld_wait();
      };
      uint32_t w[NT][4][8];
      float big[4], lu[4];
      // weights against `ref` (a masked key's scale may be anything)
      auto weigh = [&](auto mask) {
        uint64_t sum[4], nref[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          big[y] = 0.0f;
          sum[y] = f2_pack(0.0f, 0.0f);
          nref[y] = f2_pack(-ref[y], -ref[y]);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t s[2][16];
          load(q, s);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int c = 32 * q + 8 * g;
            const uint64_t ks = *reinterpret_cast<const uint64_t*>(sc + c);
            const uint64_t vs = *reinterpret_cast<const uint64_t*>(sc + KT + c);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int h = y >> 1, j = 4 * g + 2 * (y & 1);
              float d0, d1, x0, x1;
              const uint64_t kk = kScaled ? f2_mul(ks, f2_pack(qmul[y], qmul[y])) : ks;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(s[h][j]), __uint_as_float(s[h][j + 1])), kk, nref[y]), d0, d1);
              float e0 = fast_exp2(d0), e1 = fast_exp2(d1);
              f2_unpack(f2_mul(f2_pack(e0, e1), vs), x0, x1);
              if (mask) {
                if (k0 + c >= lim[y]) e0 = x0 = 0.0f;
                if (k0 + c + 1 >= lim[y]) e1 = x1 = 0.0f;
              }
              sum[y] = f2_add(sum[y], f2_pack(e0, e1));
              big[y] = max3f(big[y], fabsf(x0), fabsf(x1));
              const uint32_t hi = half_pair(x0, x1);
              w[0][2 * q + h][2 * g + (y & 1)] = hi;
              if constexpr (kSplit) w[NT - 1][2 * q + h][2 * g + (y & 1)] = half_rest(hi, x0, x1);
            }
          }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float a, b;
          f2_unpack(sum[y], a, b);
          lu[y] = l[y] + (a + b);
        }
      };
      // References move each by its own row's need only (a row that fits keeps its weights), and the
      // tile is weighed again, twice at most (infinite scores or scales never fit).  On the first try an
      // overshoot below kFarWeight says how far and rows beyond it wait; on the second, rows that still do
      // not fit ask for the maxima, as all do on the first tile.  So the way a row's reference takes, and
      // with it the rounding of its weights, depends on no other row.
      bool search = n == 0;
      for (int tries = 0;; ++tries) {
        if (!search) {
          if (masked)
            weigh(std::true_type{});
          else
            weigh(std::false_type{});
          bool need = false;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            if (lu[y] >= kMaxSum) big[y] = INFINITY;
            need = need || big[y] >= kMaxWeight;
          }
          if (tries == 2 || !__any_sync(0xffffffffu, need)) break;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            big[y] = fmaxf(big[y], __shfl_xor_sync(0xffffffffu, big[y], 1));
            big[y] = fmaxf(big[y], __shfl_xor_sync(0xffffffffu, big[y], 2));
          }
          search = tries > 0;
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y) big[y] = INFINITY;
        }
        float alpha[4];
        if (search) {
          float top[4], top_w[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) top[y] = top_w[y] = -INFINITY;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t s[2][16];
            load(q, s);
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const int c = 32 * q + 8 * g + z;
                const float ks = sc[c], lv = weight_log2(0.0f, sc[KT + c]);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const float v = __uint_as_float(s[y >> 1][4 * g + 2 * (y & 1) + z]);
                  const float x = k0 + c < lim[y] ? v * (ks * qmul[y]) : -INFINITY;
                  top[y] = fmaxf(top[y], x);
                  top_w[y] = fmaxf(top_w[y], x + lv);
                }
              }
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
#pragma unroll
            for (int x = 1; x <= 2; x <<= 1) {
              top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], x));
              top_w[y] = fmaxf(top_w[y], __shfl_xor_sync(0xffffffffu, top_w[y], x));
            }
            alpha[y] = big[y] >= kMaxWeight ? new_ref<T>(ref[y], top[y], top_w[y]) : ref[y];
          }
        } else {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            alpha[y] = big[y] >= kMaxWeight && big[y] < kFarWeight ? ref[y] + __log2f(big[y]) - kTarget<T> : ref[y];
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float moved = alpha[y];
          alpha[y] = fast_exp2(ref[y] - moved);
          ref[y] = moved;
          l[y] *= alpha[y];
        }
        search = false;
        if (n > 0) {  // O *= alpha, once the stream's previous product is in it
          ok = __all_sync(0xffffffffu, mbar_wait(&o_full[sm], (n - 1) & 1, abort_flag, p.status, kDevTimeoutSoftmax));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < DH; c += 32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t r[16];
              tmem_ld_16x256b_x4(to + h * kHalf + c, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j)
                r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha[2 * h + ((j >> 1) & 1)]);
              tmem_st_16x256b_x4(to + h * kHalf + c, r);
            }
          }
          tmem_st_wait();  // a second try reads O again
        }
      }
      if (!ok) break;
#pragma unroll
      for (int y = 0; y < 4; ++y) l[y] = lu[y];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 4; ++h)
          tmem_st_16x128b_x4(ts + (h & 1) * kHalf + x * (KT / 2) + (h >> 1) * 16, w[x][h]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&w_full[buf]);
    }
    if (ok && n > 0)
      __all_sync(0xffffffffu, mbar_wait(&o_full[sm], (n - 1) & 1, abort_flag, p.status, kDevTimeoutSoftmax));
    tc_fence_after();
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
      l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
      if (c4 == 0) {
        s_ref[sm * kRows + row0 + 8 * y] = ref[y];
        s_l[sm * kRows + row0 + 8 * y] = l[y];
      }
    }
  }
  __syncthreads();  // every product is done: Q and the ring are free

  // ---- stream B's result into shared memory, 16-byte pieces XORed with the row
  float* s_out = reinterpret_cast<float*>(smem);
  auto piece = [&](int row, int c) { return s_out + row * DH + ((c ^ (row & 7)) << 2); };
  const bool two = n_mine > 1;
  if (two && warp >= 4 && warp < 8) {
    const int row = threadIdx.x & 127;
    const uint32_t to = tbase + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::kO + DH;
#pragma unroll 1
    for (int c = 0; c < DH; c += 32) {
      uint32_t r[32];
      tmem_ld_32x32b_x32(to + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint4*>(piece(row, c / 4 + j)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
    }
  }
  __syncthreads();
  // ---- A and B join (thread = row)
  const bool alone = p.C == 1;
  if (warp < 4) {
    const int row = threadIdx.x;
    const uint32_t to = tbase + (static_cast<uint32_t>(warp * 32) << 16) + C::kO;
    float M = s_ref[row], fa = 1.0f, fb = 0.0f, L = s_l[row];
    if (two) {
      const float ra = M, rb = s_ref[kRows + row];
      M = fmaxf(ra, rb);
      fa = fast_exp2(ra - M);
      fb = fast_exp2(rb - M);
      L = fmaf(fa, L, fb * s_l[kRows + row]);
    }
    const bool in = tile.r0 + row <= tile.last;
    T* dst = tile.out_row<T>(p, in ? tile.r0 + row : 0, DH);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll 1
    for (int c = 0; c < DH; c += 32) {
      float v[32];
      uint32_t r[32];
      if (n_mine > 0) {
        tmem_ld_32x32b_x32(to + c, r);
        tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = n_mine > 0 ? __uint_as_float(r[j]) : 0.0f;
      if (two) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 o = *reinterpret_cast<const float4*>(piece(row, c / 4 + j));
          const float w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int z = 0; z < 4; ++z) v[4 * j + z] = fmaf(fa, v[4 * j + z], fb * w[z]);
        }
      }
      if (alone) {
        if (in) {
#pragma unroll
          for (int j = 0; j < 32 / kPer; ++j) {
            Vec<T, kPer> o;
#pragma unroll
            for (int z = 0; z < kPer; ++z) o.v[z] = from_f<T>(L == 0.0f ? 0.0f : v[j * kPer + z] * inv);
            reinterpret_cast<Vec<T, kPer>*>(dst + c)[j] = o;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4*>(piece(row, c / 4 + j)) =
              make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      }
    }
    if (!alone) {
      s_ref[row] = M;
      s_l[row] = L;
    }
  }
  if (!alone) {
    // ---- the cluster's CTAs join, each for its share of the tile
    cluster_sync_all();
    const int n_rows = tile.last - tile.r0 + 1;
    for (int i = rank * kTcThreads + static_cast<int>(threadIdx.x); i < n_rows * DH; i += p.C * kTcThreads) {
      const int row = i / DH, d = i % DH;
      const uint32_t a_o = smem_u32(piece(row, d >> 2) + (d & 3));
      const uint32_t a_m = smem_u32(&s_ref[row]), a_l = smem_u32(&s_l[row]);
      float M = -INFINITY;
      for (int c = 0; c < p.C; ++c) M = fmaxf(M, ld_dsmem(a_m, c));
      float acc = 0.0f, L = 0.0f;
      for (int c = 0; c < p.C; ++c) {
        const float f = fast_exp2(ld_dsmem(a_m, c) - M);
        acc = fmaf(f, ld_dsmem(a_o, c), acc);
        L = fmaf(f, ld_dsmem(a_l, c), L);
      }
      tile.out_row<T>(p, tile.r0 + row, DH)[d] = from_f<T>(L == 0.0f ? 0.0f : acc / L);
    }
    cluster_sync_all();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) drain_sleep(200000);
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

}  // namespace

template <typename T, int DH>
int attn_kv_tc(const AttnKvParams& given, cudaStream_t s) {
  using C = TcCfg<DH, sizeof(T) == 4>;
  AttnKvParams p = given;
  static bool done[64] = {false};
  int dev = 0;
  DLM_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !done[dev]) {
    DLM_CHECK_CUDA(cudaFuncSetAttribute(attn_kv_tc_kernel<T, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kWholeSm));
    if (dev < 64) done[dev] = true;
  }
  const long long row_tiles = (static_cast<long long>(p.Sq) * p.g + kRows - 1) / kRows;
  const long long tiles = row_tiles * p.B * p.Hkv;
  DLM_REQUIRE(tiles < (1ll << 27), DLM_ERR_UNSUPPORTED, "attention_kv_i8: too many rows");
  p.row_tiles = static_cast<int>(row_tiles);
  p.tiles = static_cast<int>(tiles);
  // CTAs per cluster: waves (one CTA per SM) times the longest row's keys, plus each CTA's fixed work
  // (about as long as kFixed keys), is least
  constexpr double kFixed = 512.0;
  const int sms = num_sms();
  double best = 1e30;
  for (int c = 1; c <= 8; ++c) {
    const long long units = (p.Lmax + static_cast<long long>(KT) * c - 1) / (KT * c);
    const double t = static_cast<double>((tiles * c + sms - 1) / sms) *
                     (static_cast<double>(units * KT) + kFixed);
    if (t < 0.97 * best) {
      best = t;
      p.C = c;
    }
  }
  const int smem = p.C > 1 ? kWholeSm : C::kSmem;
  DLM_CHECK_CUDA(launch_clusters(attn_kv_tc_kernel<T, DH>, static_cast<unsigned>(tiles * p.C), kTcThreads, smem, p.C,
                                 s, p));
  return DLM_OK;
}

template int attn_kv_tc<float, 64>(const AttnKvParams&, cudaStream_t);
template int attn_kv_tc<float, 128>(const AttnKvParams&, cudaStream_t);
template int attn_kv_tc<__half, 64>(const AttnKvParams&, cudaStream_t);
template int attn_kv_tc<__half, 128>(const AttnKvParams&, cudaStream_t);
template int attn_kv_tc<__nv_bfloat16, 64>(const AttnKvParams&, cudaStream_t);
template int attn_kv_tc<__nv_bfloat16, 128>(const AttnKvParams&, cudaStream_t);

}  // namespace dlm
