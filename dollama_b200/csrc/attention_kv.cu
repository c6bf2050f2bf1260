// Attention over the int8 K/V cache (kv_i8.cu): softmax(scale q k^T) v for single new tokens and
// for prompt chunks, with heads that share keys (Hq a multiple of Hkv).
//
//   s_ij = scale * kscale_j * sum_d q_id kq_jd        visible: j < kv_len and (causal) j <= pos_i,
//   p_ij = exp(s_ij - max_j s_ij)                     pos_i = kv_len - q_len + i
//   out_id = sum_j p_ij vscale_j vq_jd / sum_j p_ij   (no visible key: zeros)
//
// The g = Hq / Hkv heads of one kv head times the queries of one sequence are the rows of one
// problem (row r: query r / g, head r % g), so a key is read once for all of them.
//
// A cluster of C CTAs takes 8 NR rows of one (sequence, kv head); its CTAs' warps take 32 keys at a
// time in turn, each with its own running maximum and sum (one pass over the cache), and the
// partial results meet in shared memory: the warps' in their CTA, the CTAs' over the cluster, in a
// fixed order.  A warp's keys arrive through its own ring of asynchronous copies (16-byte pieces
// XORed with the row, so that both operands' reads are free of bank conflicts).
//
// Both products are transposed (keys, then channels, are the matrix instruction's 16 rows; the
// queries its 8 columns), so that a few rows waste little, and their A operands come straight from
// the codes: which k index of a fragment stands for which d (or key) is free as long as both
// operands agree, so a lane takes 16 consecutive bytes of a key, and for V the same 8 (16) channels
// of four keys.  An int8 code becomes an fp16 value exactly (0x6400 | (code + 128) is 1152 + code).
// The scales stay outside the products: kscale multiplies the finished dot product; vscale
// multiplies p in fp32.
//
// Precision: q is exact in fp16 for fp16, scaled per row by a power of two to [2^14, 2^15) for bf16
// (exact down to 2^-25 of the row's maximum) and split into two fp16 terms for fp32.  The weights
// w_ij = p_ij vscale_j are taken against a reference of their row's own that keeps them in fp16's
// range (so a key that a row does not see has no part in it) and rounded to fp16 (a relative error of
// 2^-11 each), for fp32 split into two terms.  Sums are fp32.
//
// Bound by the cache's bytes once they are many: 64 sequences of up to 16384 tokens, 32 heads on 8, Dh
// 128, fp16: 247-254 us, all of the measured copy rate; 8 of them 41 us (77 %: the start, the joins and
// uneven lengths take 10).  A form with the queries as the instruction's 16 rows and loads straight into
// fragments took 191 us there: half-empty tiles, and no loads in flight under the arithmetic.
#include "attention_kv.cuh"

namespace dlm {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 32;  // keys a warp takes at a time

// NR: tiles of 8 rows; ST: units of a warp's ring (the copies in flight), more of them where the grid
// leaves an SM one CTA: with two, a warp that takes 16 units of one sequence's keys waits for each.
template <int DH, int NR, int ST>
struct Cfg {
  static constexpr int kStage = kUnit * (2 * DH + 8);  // K, V codes, two scales
  static constexpr int kWarpBytes = ST * kStage;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static_assert(kWarpBytes >= 8 * NR * DH * 4, "a warp's partial result reuses its ring");
};
template <int DH>
constexpr int kShallow = DH == 64 ? 3 : 2;
template <int DH>
constexpr int kDeep = DH == 64 ? 8 : 5;
constexpr int kMaxCluster = 8;

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async4(void* dst_smem, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst_smem)), "l"(src), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// byte of 16-byte piece `ch` of key row `r` in a staged [32][DH] block
template <int DH>
__device__ __forceinline__ int swz(int r, int ch) {
  if constexpr (DH == 128) return r * 128 + ((ch ^ (r & 6) ^ ((r & 1) << 2)) << 4);
  const int m = r >> 1;
  return m * 128 + (((r ^ m) & 1) << 6) + ((ch ^ (m & 2)) << 4);
}

template <typename T, int DH, int NR, int ST, bool kSolo>
__global__ void __launch_bounds__(kThreads)
    attn_kv_kernel(const AttnKvParams p) {
  using C = Cfg<DH, NR, ST>;
  constexpr int kRows = 8 * NR;
  constexpr bool kSplit = sizeof(T) == 4;                    // two fp16 terms for q and the weights
  constexpr bool kScaled = !std::is_same<T, __half>::value;  // q scaled into fp16's range
  constexpr int NT = kSplit ? 2 : 1;
  constexpr int KS = DH / 16;  // k-steps of q.k, and channel tiles of p.v
  constexpr int DJ = DH / 8;   // channels of a lane
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ float s_cm[kRows], s_cl[kRows];
  extern __shared__ __align__(128) uint8_t s_ring[];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, c4 = lane & 3;
  const int rank = kSolo ? 0 : static_cast<int>(blockIdx.x % p.C);
  const int t = kSolo ? static_cast<int>(blockIdx.x) * kWarps + warp : static_cast<int>(blockIdx.x / p.C);
  if (kSolo && t >= p.tiles) return;  // (a lone warp meets no barrier)
  const AttnKvTile tile(p, t, kRows, (kSolo ? lane : threadIdx.x) == 0);
  const int r0 = tile.r0, last = tile.last, n_keys = tile.n_keys, n_all = tile.n_all;
  int lim[NR][2];                                // of rows 2 c4 and 2 c4 + 1
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int r = r0 + 8 * n + 2 * c4 + z;
      lim[n][z] = r <= last ? tile.seen(p, r) : n_keys;
    }

  const size_t head = tile.head(p);
  const int8_t* kb = p.kq + head * p.Lmax * DH;
  const int8_t* vb = p.vq + head * p.Lmax * DH;
  const float* ksb = p.ks + head * p.Lmax;
  const float* vsb = p.vs + head * p.Lmax;
  uint8_t* ring = s_ring + warp * C::kWarpBytes;
  const int first = kSolo ? 0 : (rank * kWarps + warp) * kUnit, stride = kSolo ? kUnit : p.C * kWarps * kUnit;

  // keys k0 .. k0 + 31 into stage st (zeros beyond n_keys): piece i * 32 + lane is bytes 16 lane ..
  // of rows i * kRowsPer .., and its place repeats every 8 rows
  constexpr int kPieces = DH / 16, kRowsPer = 32 / kPieces, kPeriod = 8 / kRowsPer;
  int dst_off[kPeriod];
#pragma unroll
  for (int i = 0; i < kPeriod; ++i) dst_off[i] = swz<DH>(i * kRowsPer + lane / kPieces, lane % kPieces);
  auto fetch = [&](int k0, int st) {
    uint8_t* dst = ring + st * C::kStage;
    if (k0 + kUnit <= n_keys) {
      const int8_t* k = kb + static_cast<size_t>(k0) * DH + 16 * lane;
      const int8_t* v = vb + static_cast<size_t>(k0) * DH + 16 * lane;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        uint8_t* d = dst + dst_off[i % kPeriod] + (i / kPeriod) * 8 * DH;
        cp_async16(d, k + i * 512, 16);
        cp_async16(d + kUnit * DH, v + i * 512, 16);
      }
      cp_async4(dst + 2 * kUnit * DH + 4 * lane, ksb + k0 + lane, 4);
      cp_async4(dst + 2 * kUnit * DH + 4 * (kUnit + lane), vsb + k0 + lane, 4);
    } else if (k0 < n_keys) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const bool in = k0 + i * kRowsPer + lane / kPieces < n_keys;
        const size_t off = in ? static_cast<size_t>(k0) * DH + i * 512 + 16 * lane : 0;
        uint8_t* d = dst + dst_off[i % kPeriod] + (i / kPeriod) * 8 * DH;
        cp_async16(d, kb + off, in ? 16u : 0u);
        cp_async16(d + kUnit * DH, vb + off, in ? 16u : 0u);
      }
      const bool in = k0 + lane < n_keys;
      const size_t off = in ? k0 + lane : 0;
      cp_async4(dst + 2 * kUnit * DH + 4 * lane, ksb + off, in ? 4u : 0u);
      cp_async4(dst + 2 * kUnit * DH + 4 * (kUnit + lane), vsb + off, in ? 4u : 0u);
    }
    cp_async_commit();
  };
  int k_next = first;
  for (int i = 0; i < ST - 1; ++i, k_next += stride) fetch(k_next, i);

  // ---- q, the B operand: row gr, channels 64 h + 16 c4 + 4 z + {0, 1 | 2, 3} in k-step 4 h + z
  uint32_t qf[NT][NR][KS][2];
  float qmul[NR][2];  // of rows 2 c4 and 2 c4 + 1
  {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = r0 + 8 * n + gr;
      float f[KS * 4];
      if (r <= last) {
        const T* src = tile.q_row<T>(p, r, DH);
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) f[i] = to_f(src[(i >> 4) * 64 + 16 * c4 + (i & 15)]);
      } else {
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) f[i] = 0.0f;
      }
      float up = 1.0f, mul = p.scale_log2;
      if constexpr (kScaled) {
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) mx = fmaxf(mx, fabsf(f[i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = q_up(mx);
        up = pow2i(e);
        mul = p.scale_log2 * pow2i(-e);
      }
      qmul[n][0] = __shfl_sync(0xffffffffu, mul, 8 * c4);  // lane 4 r holds row r
      qmul[n][1] = __shfl_sync(0xffffffffu, mul, 8 * c4 + 4);
#pragma unroll
      for (int i = 0; i < KS * 2; ++i) {
        const float a0 = f[2 * i] * up, a1 = f[2 * i + 1] * up;
        qf[0][n][i >> 1][i & 1] = half_pair(a0, a1);
        if constexpr (kSplit) qf[NT - 1][n][i >> 1][i & 1] = half_rest(qf[0][n][i >> 1][i & 1], a0, a1);
      }
    }
  }

  // o: channels gr * DJ + 2 j + {0: [0..1], 1: [2..3]} of rows 2 c4 + {0, 1}
  float o[NR][KS][4], ref[NR][2], l[NR][2];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][j][i] = 0.0f;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      ref[n][z] = kNoRef;
      l[n][z] = 0.0f;
    }
  }

  // this lane's pieces: key row gr, channels 64 h + 16 c4; value rows 2 c4 and 2 c4 + 1, channels
  // gr * DJ (the places repeat every 8 rows)
  int k_off[DH / 64], v_off[2];
#pragma unroll
  for (int h = 0; h < DH / 64; ++h) k_off[h] = swz<DH>(gr, 4 * h + c4);
#pragma unroll
  for (int i = 0; i < 2; ++i) v_off[i] = kUnit * DH + swz<DH>(2 * c4 + i, gr * DJ / 16) + (gr * DJ) % 16;

  int st = 0;
  for (int k0 = first; k0 < n_keys; k0 += stride, k_next += stride) {
    fetch(k_next, st == 0 ? ST - 1 : st - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
    __syncwarp();
    const uint8_t* sk = ring + st * C::kStage;
    const float* sks = reinterpret_cast<const float*>(sk + 2 * kUnit * DH) + gr;
    // ---- scores: keys 16 t + gr + {0: [0..1], 8: [2..3]} of rows 2 c4 + {0, 1}
    float s[2][NR][4];
    float ksc[2][2], vsc[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[u][n][j] = 0.0f;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h) {
        const uint4 w0 = *reinterpret_cast<const uint4*>(sk + k_off[h] + 16 * u * DH);
        const uint4 w1 = *reinterpret_cast<const uint4*>(sk + k_off[h] + (16 * u + 8) * DH);
        const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const uint32_t y0 = x0[z] ^ 0x80808080u, y1 = x1[z] ^ 0x80808080u;
          const uint32_t a[4] = {code_pair(y0, 0x4140), code_pair(y1, 0x4140), code_pair(y0, 0x4342),
                                 code_pair(y1, 0x4342)};
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int k = 0; k < NT; ++k) mma_f16(s[u][n], a, qf[k][n][4 * h + z][0], qf[k][n][4 * h + z][1]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ksc[u][h] = sks[16 * u + 8 * h];
        vsc[u][h] = sks[kUnit + 16 * u + 8 * h];
      }
    }
    // weights against the references so far (a masked key's scale may be anything)
    const bool masked = k0 + kUnit > n_all;
    float w[2][NR][4], lu[NR][2], big = 0.0f, sum = 0.0f;
    auto weigh = [&](auto mask) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          lu[n][z] = l[n][z];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int i = 2 * h + z;
              const bool hidden = mask && k0 + 16 * u + gr + 8 * h >= lim[n][z];
              const float d = fmaf(s[u][n][i], ksc[u][h] * qmul[n][z], -ref[n][z]);
              const float e = hidden ? 0.0f : fast_exp2(d);
              lu[n][z] += e;
              w[u][n][i] = hidden ? 0.0f : e * vsc[u][h];
            }
            big = max3f(big, fabsf(w[u][n][z]), fabsf(w[u][n][2 + z]));
          }
          sum = fmaxf(sum, lu[n][z]);
        }
    };
    if (masked)
      weigh(std::true_type{});
    else
      weigh(std::false_type{});
    if (__any_sync(0xffffffffu, big >= kMaxWeight || sum >= kMaxSum)) {
      // the references move (the first unit, a score well above those so far, a large vscale), each by
      // its own row's need only; a row that stays keeps the weights it has (formed again as below they
      // would differ by a rounding): no row's result depends on its neighbours, to the bit
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float top = -INFINITY, top_w = -INFINITY, most = lu[n][z] >= kMaxSum ? INFINITY : 0.0f;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              most = fmaxf(most, fabsf(w[u][n][2 * h + z]));
              float& x = s[u][n][2 * h + z];
              x *= ksc[u][h] * qmul[n][z];
              if (k0 + 16 * u + gr + 8 * h >= lim[n][z]) x = -INFINITY;
              top = fmaxf(top, x);
              top_w = fmaxf(top_w, weight_log2(x, vsc[u][h]));
            }
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            top_w = fmaxf(top_w, __shfl_xor_sync(0xffffffffu, top_w, x));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
          }
          const bool moves = most >= kMaxWeight;
          const float to = moves ? new_ref<T>(ref[n][z], top, top_w) : ref[n][z];
          const float alpha = fast_exp2(ref[n][z] - to);
          ref[n][z] = to;
          float lm = l[n][z] * alpha;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float e = fast_exp2(s[u][n][2 * h + z] - to);
              const float wm = k0 + 16 * u + gr + 8 * h >= lim[n][z] ? 0.0f : e * vsc[u][h];
              lm += e;
              if (moves) w[u][n][2 * h + z] = wm;
            }
          if (moves) lu[n][z] = lm;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            o[n][j][z] *= alpha;
            o[n][j][2 + z] *= alpha;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      l[n][0] = lu[n][0];
      l[n][1] = lu[n][1];
    }
    // ---- the weights as the B operand of p.v: [key][row] tiles transposed to [row][key]
    uint32_t pf[NT][NR][2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w0 = w[u][n][2 * h], w1 = w[u][n][2 * h + 1];
          const uint32_t hi = half_pair(w0, w1);
          pf[0][n][u][h] = transpose8x8(hi);
          if constexpr (kSplit) pf[NT - 1][n][u][h] = transpose8x8(half_rest(hi, w0, w1));
        }
    // ---- p.v: channels gr * DJ .. + DJ - 1 of keys 16 u + 2 c4 + {0, 1, 8, 9}
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Vec<uint32_t, DJ / 4> vw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* src = sk + v_off[i & 1] + (16 * u + (i >> 1) * 8) * DH;
        vw[i] = *reinterpret_cast<const Vec<uint32_t, DJ / 4>*>(src);
      }
#pragma unroll
      for (int z = 0; z < DJ / 4; ++z) {
        const uint32_t w0 = vw[0].v[z] ^ 0x80808080u, w1 = vw[1].v[z] ^ 0x80808080u;
        const uint32_t w2 = vw[2].v[z] ^ 0x80808080u, w3 = vw[3].v[z] ^ 0x80808080u;
#pragma unroll
        for (int y = 0; y < 2; ++y) {  // channels 4 z + 2 y + {0, 1}
          const uint32_t x01 = __byte_perm(w0, w1, y ? 0x7362 : 0x5140);
          const uint32_t x23 = __byte_perm(w2, w3, y ? 0x7362 : 0x5140);
          const uint32_t a[4] = {code_pair(x01, 0x4140), code_pair(x01, 0x4342), code_pair(x23, 0x4140),
                                 code_pair(x23, 0x4342)};
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int k = 0; k < NT; ++k) mma_f16(o[n][2 * z + y], a, pf[k][n][u][0], pf[k][n][u][1]);
        }
      }
    }
    if (++st == ST) st = 0;
    __syncwarp();  // every lane is done with the stage before its next fetch
  }
  cp_async_wait_all();
  __syncwarp();

  if constexpr (kSolo) {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) l[n][z] += __shfl_xor_sync(0xffffffffu, l[n][z], x);
        const int r = 8 * n + 2 * c4 + z;
        if (r0 + r > last) continue;
        const float down = l[n][z] == 0.0f ? 0.0f : 1.0f / l[n][z];
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
        Vec<T, kPer> v[DJ / kPer];
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          v[2 * j / kPer].v[2 * j % kPer] = from_f<T>(o[n][j][z] * down);
          v[(2 * j + 1) / kPer].v[(2 * j + 1) % kPer] = from_f<T>(o[n][j][2 + z] * down);
        }
        T* dst = tile.out_row<T>(p, r0 + r, DH) + gr * DJ;
#pragma unroll
        for (int j = 0; j < DJ / kPer; ++j) reinterpret_cast<Vec<T, kPer>*>(dst)[j] = v[j];
      }
    return;
  }
  // ---- this warp's partial results: reference, sum and o, into its ring
  float* s_o = reinterpret_cast<float*>(ring);  // [kRows][DH]
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) l[n][z] += __shfl_xor_sync(0xffffffffu, l[n][z], x);
      const int r = 8 * n + 2 * c4 + z;
      if (gr == 0) {
        s_m[warp][r] = ref[n][z];
        s_l[warp][r] = l[n][z];
      }
#pragma unroll
      for (int j = 0; j < KS; j += 2)
        *reinterpret_cast<float4*>(s_o + r * DH + gr * DJ + 2 * j) =
            make_float4(o[n][j][z], o[n][j][2 + z], o[n][j + 1][z], o[n][j + 1][2 + z]);
    }
  __syncthreads();
  // ---- the CTA's warps join, element by element (each read and written by one thread)
  s_o = reinterpret_cast<float*>(s_ring);
  constexpr int kWarpFloats = C::kWarpBytes / 4;
  const int n_rows = last - r0 + 1;  // rows of this tile that exist
  for (int i = threadIdx.x; i < n_rows * DH; i += kThreads) {
    const int r = i / DH;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
    float acc = 0.0f, ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(s_m[w][r] - M);
      acc = fmaf(f, s_o[w * kWarpFloats + i], acc);
      ls = fmaf(f, s_l[w][r], ls);
    }
    if (p.C == 1) {
      tile.out_row<T>(p, r0 + r, DH)[i % DH] = from_f<T>(ls == 0.0f ? 0.0f : acc / ls);
      continue;
    }
    s_o[i] = acc;
    if (i % DH == 0) {
      s_cm[r] = M;
      s_cl[r] = ls;
    }
  }
  if (p.C == 1) return;
  cluster_sync_all();
  for (int i = rank * kThreads + threadIdx.x; i < n_rows * DH; i += p.C * kThreads) {
    const int r = i / DH;
    // every CTA's three values are requested before any is used
    float m[kMaxCluster], l[kMaxCluster], v[kMaxCluster], M = kNoRef, acc = 0.0f, L = 0.0f;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < p.C) {
        m[c] = ld_dsmem(smem_u32(&s_cm[r]), c);
        l[c] = ld_dsmem(smem_u32(&s_cl[r]), c);
        v[c] = ld_dsmem(smem_u32(&s_o[i]), c);
      }
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < p.C) M = fmaxf(M, m[c]);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < p.C) {
        const float f = fast_exp2(m[c] - M);
        acc = fmaf(f, v[c], acc);
        L = fmaf(f, l[c], L);
      }
    tile.out_row<T>(p, r0 + r, DH)[i % DH] = from_f<T>(L == 0.0f ? 0.0f : acc / L);
  }
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// Raises the kernel's shared-memory limit and finds how many CTAs an SM holds, once per device.
template <typename K>
int residency(K kernel, int smem, int (&cache)[64], int& per_sm) {
  int dev = 0;
  DLM_CHECK_CUDA(cudaGetDevice(&dev));
  per_sm = dev < 64 ? cache[dev] : 0;
  if (per_sm > 0) return DLM_OK;
  DLM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  DLM_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, smem));
  if (per_sm < 1) per_sm = 1;
  if (dev < 64) cache[dev] = per_sm;
  return DLM_OK;
}

template <typename T, int DH, int NR>
int launch(AttnKvParams p, cudaStream_t s) {
  using Few = Cfg<DH, NR, kDeep<DH>>;
  using Many = Cfg<DH, NR, kShallow<DH>>;
  auto many = attn_kv_kernel<T, DH, NR, kShallow<DH>, false>;
  auto few = attn_kv_kernel<T, DH, NR, kDeep<DH>, false>;
  auto solo = attn_kv_kernel<T, DH, NR, kShallow<DH>, true>;
  static int cache[3][64] = {{0}};
  int per_many = 0, per_few = 0, per_solo = 0;
  int rc = residency(many, Many::kSmem, cache[0], per_many);
  if (rc == DLM_OK) rc = residency(few, Few::kSmem, cache[1], per_few);
  if (rc == DLM_OK) rc = residency(solo, Many::kSmem, cache[2], per_solo);
  if (rc != DLM_OK) return rc;
  const long long row_tiles = (static_cast<long long>(p.Sq) * p.g + 8 * NR - 1) / (8 * NR);
  const long long tiles = row_tiles * p.B * p.Hkv;
  DLM_REQUIRE(tiles < (1ll << 26), DLM_ERR_UNSUPPORTED, "attention_kv_i8: too many rows");
  p.row_tiles = static_cast<int>(row_tiles);
  p.tiles = static_cast<int>(tiles);
  // Waves times keys of a warp (plus its fixed work, about as long as kFixed keys), for one warp per
  // tile and for clusters of 1 to 8 CTAs per tile (a cluster of 16, which needs
  // the kernel's leave, cost 7 us more to launch than it saved).
  constexpr double kFixed = 100.0;
  const int sms = num_sms();
  auto cost = [&](long long ctas, int resident, int warps) {
    const long long slots = static_cast<long long>(resident) * sms;
    const long long units = (p.Lmax + static_cast<long long>(kUnit) * warps - 1) / (kUnit * warps);
    return static_cast<double>((ctas + slots - 1) / slots) * (static_cast<double>(units * kUnit) + kFixed);
  };
  const long long solo_ctas = (tiles + kWarps - 1) / kWarps;
  double best = cost(solo_ctas, per_solo, 1);
  p.C = 0;
  for (int c = 1; c <= kMaxCluster; ++c) {
    const double t = cost(tiles * c, per_many, c * kWarps);
    if (t < 0.97 * best) {
      best = t;
      p.C = c;
    }
  }
  if (p.C == 0) {
    DLM_CHECK_CUDA(launch_pdl(solo, dim3(static_cast<unsigned>(solo_ctas)), dim3(kThreads), Many::kSmem, s, p));
    return DLM_OK;
  }
  const unsigned grid = static_cast<unsigned>(tiles * p.C);
  if (static_cast<long long>(grid) <= static_cast<long long>(per_few) * sms)
    DLM_CHECK_CUDA(launch_clusters(few, grid, kThreads, Few::kSmem, p.C, s, p));
  else
    DLM_CHECK_CUDA(launch_clusters(many, grid, kThreads, Many::kSmem, p.C, s, p));
  return DLM_OK;
}

template <typename T, int DH>
int launch_rows(const AttnKvParams& p, cudaStream_t s) {
  const long long rows = static_cast<long long>(p.Sq) * p.g;
  if (rows <= 8) return launch<T, DH, 1>(p, s);
  if (rows <= kAttnKvFewRows) return launch<T, DH, 2>(p, s);
  return attn_kv_tc<T, DH>(p, s);
}

}  // namespace

}  // namespace dlm

extern "C" int dlm_attention_kv_i8(const void* q, int ldq, const int8_t* kq, const float* kscale,
                                   const int8_t* vq, const float* vscale, void* out, int ldo, int B, int Hq,
                                   int Hkv, int Sq, int Dh, int Lmax, const int* kv_len, const int* q_len,
                                   int causal, float scale, int dtype, void* stream) {
  using namespace dlm;
  DLM_REQUIRE(B >= 0 && Hq >= 0 && Hkv >= 0 && Sq >= 0 && Lmax >= 0, DLM_ERR_INVALID,
              "attention_kv_i8: negative size");
  DLM_REQUIRE(dtype_ok(dtype), DLM_ERR_INVALID, "attention_kv_i8: unknown dtype %d", dtype);
  DLM_REQUIRE(Dh == 64 || Dh == 128, DLM_ERR_UNSUPPORTED, "attention_kv_i8: head dim %d (64 or 128)", Dh);
  if (B == 0 || Hq == 0 || Sq == 0) return DLM_OK;
  DLM_REQUIRE(Hkv > 0 && Hq % Hkv == 0, DLM_ERR_INVALID, "attention_kv_i8: Hq=%d is no multiple of Hkv=%d", Hq,
              Hkv);
  DLM_REQUIRE(q && out && kv_len && (Lmax == 0 || (kq && kscale && vq && vscale)), DLM_ERR_INVALID,
              "attention_kv_i8: null pointer");
  const long long width = static_cast<long long>(Hq) * Dh;
  DLM_REQUIRE(ldq >= width && ldo >= width, DLM_ERR_INVALID,
              "attention_kv_i8: a token stride is below Hq * Dh = %lld", width);
  const int vec = static_cast<int>(16 / dtype_size(dtype));
  DLM_REQUIRE(aligned16(q) && aligned16(out) && ldq % vec == 0 && ldo % vec == 0, DLM_ERR_INVALID,
              "attention_kv_i8: q / out rows must start on 16-byte boundaries");
  DLM_REQUIRE(aligned16(kq) && aligned16(vq), DLM_ERR_INVALID,
              "attention_kv_i8: cache codes must be 16-byte aligned");
  DLM_REQUIRE(aligned4(kscale) && aligned4(vscale) && aligned4(kv_len) && aligned4(q_len), DLM_ERR_INVALID,
              "attention_kv_i8: a scale or length array is not 4-byte aligned");
  DLM_REQUIRE(scale > -INFINITY && scale < INFINITY, DLM_ERR_INVALID, "attention_kv_i8: scale is not finite");
  const int g = Hq / Hkv;
  DLM_REQUIRE(static_cast<long long>(Sq) * g < (1ll << 30) && Lmax <= (1 << 30), DLM_ERR_UNSUPPORTED,
              "attention_kv_i8: too many rows or cache positions");
  const AttnKvParams p{q, kq, kscale, vq, vscale, out, kv_len, q_len, ldq, ldo, B, Hq, Hkv, Sq, Lmax, g,
                       1, 1, causal, 1, scale * 1.4426950408889634f, device_status_ptr(),
                       device_position_ptr()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    if (Dh == 64) return launch_rows<T, 64>(p, s);
    return launch_rows<T, 128>(p, s);
  });
}
