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
// One cluster of C CTAs takes 16 rows of one (sequence, kv head); its CTAs' warps take 32 keys at a
// time in turn, each with its own running maximum and sum (one pass over the cache), and the
// partial results meet in shared memory: the warps' in their CTA, the CTAs' over the cluster, in a
// fixed order.  Codes go from global memory straight into matrix-instruction fragments: which k
// index of a fragment stands for which d (or key) is free as long as both operands agree, so a
// lane takes 16 consecutive bytes of a key, and for V the same 8 (16) channels of four keys.  An
// int8 code becomes an fp16 value exactly (0x6400 | (code + 128) is 1152 + code).  The scales stay
// outside the products: kscale multiplies the finished dot product; vscale multiplies p in fp32.
//
// Precision: q is exact in fp16 for fp16, scaled per row by a power of two to [2^14, 2^15) for bf16
// (exact down to 2^-25 of the row's maximum) and split into two fp16 terms for fp32.  The weights
// w_ij = p_ij vscale_j are scaled by a power of two that follows the row's largest one, to [2^14,
// 2^15), and rounded to fp16 (a relative error of 2^-11 each, down to 2^-29 of the largest), for
// fp32 split into two terms; each row has its own scale, so a key that a row does not see has no
// part in it.  Sums are fp32.
#include <cfloat>
#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;   // rows of one tile
constexpr int kUnit = 32;   // keys a warp takes at a time

struct AttnKvParams {
  const void* q;
  const int8_t* kq;
  const float* ks;
  const int8_t* vq;
  const float* vs;
  void* out;
  const int* kv_len;
  const int* q_len;
  long long ldq, ldo;
  int B, Hq, Hkv, Sq, Lmax, g, row_tiles, causal, C;
  float scale_log2;
  int* status;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t code_pair(uint32_t biased, uint32_t sel) {
  // two biased codes (code + 128) picked by sel -> fp16 pair of the codes
  const uint32_t h = __byte_perm(biased, 0x64646464u, sel);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1152.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^e as a float for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// smallest e with |x| < 2^e for a normal x (the biased exponent alone)
__device__ __forceinline__ int exp_above(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 0xFF) - 126; }

__device__ __forceinline__ float ld_dsmem(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n"
      ".reg .b32 ra;\n"
      "mapa.shared::cluster.u32 ra, %1, %2;\n"
      "ld.shared::cluster.f32 %0, [ra];\n"
      "}\n"
      : "=f"(v)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

template <typename T, int DH>
__global__ void __launch_bounds__(kThreads)
    attn_kv_kernel(const AttnKvParams p) {
  constexpr bool kSplit = sizeof(T) == 4;                    // two fp16 terms for q and p
  constexpr bool kScaled = !std::is_same<T, __half>::value;  // q scaled into fp16's range
  constexpr int NT = kSplit ? 2 : 1;
  constexpr int KS = DH / 16;   // k-steps of q.k
  constexpr int DJ = DH / 8;    // channel tiles of p.v
  griddep_wait();  // inputs come from the previous kernel (programmatic dependent launch)
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ float s_cm[kRows], s_cl[kRows];
  extern __shared__ float s_o[];  // [kWarps][kRows][DH]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gr = lane >> 2, c4 = lane & 3;
  const int rank = static_cast<int>(blockIdx.x % p.C);
  int t = static_cast<int>(blockIdx.x / p.C);
  const int rt = t % p.row_tiles;
  t /= p.row_tiles;
  const int hkv = t % p.Hkv, b = t / p.Hkv;

  int n_kv = p.kv_len[b];
  if (n_kv < 0 || n_kv > p.Lmax) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kDevBadPosition);
    n_kv = n_kv < 0 ? 0 : p.Lmax;
  }
  int n_q = p.q_len ? p.q_len[b] : p.Sq;
  n_q = n_q < 0 ? 0 : (n_q > p.Sq ? p.Sq : n_q);
  const int rows = n_q * p.g;  // rows of this (sequence, kv head)
  const int r0 = rt * kRows;
  // keys row r sees: [0, vis(r))
  auto vis = [&](int r) {
    if (r >= rows) return 0;
    if (!p.causal) return n_kv;
    const int e = n_kv - n_q + r / p.g + 1;
    return e < 0 ? 0 : e;
  };
  const int last = (r0 + kRows < rows ? r0 + kRows : rows) - 1;
  const int n_keys = last < r0 ? 0 : vis(last);  // the last row sees the most
  const int lim[2] = {vis(r0 + gr), vis(r0 + gr + 8)};

  // ---- q fragments: rows gr and gr + 8, channels 16 c4 + 4 t + {0, 1 | 2, 3} (+ 64 from k-step 4 on)
  uint32_t qf[NT][KS][4];
  float qmul[2];
  {
    const T* q = static_cast<const T*>(p.q);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + gr + 8 * h;
      float f[KS * 4];
      if (r < rows) {
        const T* src = q + (static_cast<size_t>(b) * p.Sq + r / p.g) * p.ldq +
                       (static_cast<size_t>(hkv) * p.g + r % p.g) * DH;
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) f[i] = to_f(src[(i >> 4) * 64 + 16 * c4 + (i & 15)]);
      } else {
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) f[i] = 0.0f;
      }
      float up = 1.0f;
      qmul[h] = p.scale_log2;
      if constexpr (kScaled) {
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) mx = fmaxf(mx, fabsf(f[i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = 15 - exp_above(mx);
        e = e > 100 ? 100 : e;  // rows below 2^-85: products below 2^-78 of any use
        up = pow2i(e);
        qmul[h] = p.scale_log2 * pow2i(-e);
      }
#pragma unroll
      for (int i = 0; i < KS * 2; ++i) {
        const float a0 = f[2 * i] * up, a1 = f[2 * i + 1] * up;
        const __half2 hi = __floats2half2_rn(a0, a1);
        qf[0][i >> 1][(i & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&hi);
        if constexpr (kSplit) {
          const float2 hf = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(a0 - hf.x, a1 - hf.y);
          qf[NT - 1][i >> 1][(i & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&lo);
        }
      }
    }
  }

  const size_t head = static_cast<size_t>(b) * p.Hkv + hkv;
  const int8_t* kb = p.kq + head * p.Lmax * DH;
  const int8_t* vb = p.vq + head * p.Lmax * DH;
  const float* ksb = p.ks + head * p.Lmax;
  const float* vsb = p.vs + head * p.Lmax;

  float o[DJ][4];
#pragma unroll
  for (int j = 0; j < DJ; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  // largest |weight| of each row so far (relative to m) and its exponent: o is sum w code 2^(15 - ew)
  float wm[2] = {0.0f, 0.0f};
  int ew[2] = {-100, -100};

  for (int k0 = (rank * kWarps + warp) * kUnit; k0 < n_keys; k0 += p.C * kWarps * kUnit) {
    // ---- loads: K codes of key 8 i + gr, V codes of keys 16 u + {2 c4, + 1, + 8, + 9}, scales
    uint4 kw[4][DH / 64];
    Vec<uint32_t, DH / 32> vw[2][4];
    float ksc[4][2], vsc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k0 + 8 * i + gr;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h)
        kw[i][h] = key < n_keys ? *reinterpret_cast<const uint4*>(kb + static_cast<size_t>(key) * DH + h * 64 + 16 * c4)
                                : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = k0 + 8 * i + 2 * c4 + h;
        const bool in = key < n_keys;
        ksc[i][h] = in ? ksb[key] : 0.0f;
        vsc[i][h] = in ? vsb[key] : 0.0f;
      }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = k0 + 16 * u + 2 * c4 + (i >> 1) * 8 + (i & 1);
        if (key < n_keys) {
          vw[u][i] = *reinterpret_cast<const Vec<uint32_t, DH / 32>*>(vb + static_cast<size_t>(key) * DH + gr * DJ);
        } else {
#pragma unroll
          for (int z = 0; z < DH / 32; ++z) vw[u][i].v[z] = 0;
        }
      }
    // ---- scores
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.0f;
#pragma unroll
      for (int h = 0; h < DH / 64; ++h) {
        const uint32_t w[4] = {kw[i][h].x, kw[i][h].y, kw[i][h].z, kw[i][h].w};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const uint32_t x = w[z] ^ 0x80808080u;
          const uint32_t b0 = code_pair(x, 0x4140), b1 = code_pair(x, 0x4342);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[i], qf[n][h * 4 + z], b0, b1);
        }
      }
    }
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 8 * i + 2 * c4 + (j & 1);
        s[i][j] = key < lim[j >> 1] ? s[i][j] * (ksc[i][j & 1] * qmul[j >> 1]) : -INFINITY;
        mx[j >> 1] = fmaxf(mx[j >> 1], s[i][j]);
      }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
      mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
    }
    // ---- weights: s becomes w
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mu = mx[h] == -INFINITY ? 0.0f : mx[h];  // no visible key yet
      alpha[h] = fast_exp2(m[h] - mu);
      m[h] = mx[h];
      l[h] *= alpha[h];
      wm[h] *= alpha[h];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int key = k0 + 8 * i + 2 * c4 + z;
          const float e = fast_exp2(s[i][2 * h + z] - mu);
          l[h] += e;
          // a masked key's scale may be anything
          s[i][2 * h + z] = key < lim[h] ? e * vsc[i][z] : 0.0f;
          wm[h] = fmaxf(wm[h], fabsf(s[i][2 * h + z]));
        }
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      wm[0] = fmaxf(wm[0], __shfl_xor_sync(0xffffffffu, wm[0], x));
      wm[1] = fmaxf(wm[1], __shfl_xor_sync(0xffffffffu, wm[1], x));
    }
    float up[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = max(exp_above(wm[h]), -100);
      const float a = alpha[h] * pow2i(min(max(ew[h] - e, -126), 127));
      ew[h] = e;
      up[h] = pow2i(15 - e);
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        o[j][2 * h] *= a;
        o[j][2 * h + 1] *= a;
      }
    }
    // ---- the A operand of p.v: k-step u takes key tiles 2 u and 2 u + 1
    uint32_t pf[NT][2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float w0 = s[i][2 * h] * up[h], w1 = s[i][2 * h + 1] * up[h];
        const __half2 hi = __floats2half2_rn(w0, w1);
        pf[0][i >> 1][(i & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&hi);
        if constexpr (kSplit) {
          const float2 hf = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(w0 - hf.x, w1 - hf.y);
          pf[NT - 1][i >> 1][(i & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&lo);
        }
      }
    // ---- p.v
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int z = 0; z < DH / 32; ++z) {
        const uint32_t w0 = vw[u][0].v[z] ^ 0x80808080u, w1 = vw[u][1].v[z] ^ 0x80808080u;
        const uint32_t w2 = vw[u][2].v[z] ^ 0x80808080u, w3 = vw[u][3].v[z] ^ 0x80808080u;
        const uint32_t lo01 = __byte_perm(w0, w1, 0x5140), hi01 = __byte_perm(w0, w1, 0x7362);
        const uint32_t lo23 = __byte_perm(w2, w3, 0x5140), hi23 = __byte_perm(w2, w3, 0x7362);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16(o[4 * z + 0], pf[n][u], code_pair(lo01, 0x4140), code_pair(lo23, 0x4140));
          mma_f16(o[4 * z + 1], pf[n][u], code_pair(lo01, 0x4342), code_pair(lo23, 0x4342));
          mma_f16(o[4 * z + 2], pf[n][u], code_pair(hi01, 0x4140), code_pair(hi23, 0x4140));
          mma_f16(o[4 * z + 3], pf[n][u], code_pair(hi01, 0x4342), code_pair(hi23, 0x4342));
        }
      }
  }

  // ---- this warp's partial results: maximum, sum, and o in true scale
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float down = pow2i(ew[h] - 15);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = gr + 8 * h;
    if (c4 == 0) {
      s_m[warp][r] = m[h];
      s_l[warp][r] = l[h];
    }
    float* dst = s_o + (warp * kRows + r) * DH;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int j = 0; j < DJ; ++j) dst[(2 * c4 + z) * DJ + j] = o[j][2 * h + z] * down;
  }
  __syncthreads();
  // weight of a partial result with maximum m against the joint maximum M (0 where it saw no key)
  auto weight = [](float mm, float M) { return mm == -INFINITY ? 0.0f : fast_exp2(mm - M); };
  // ---- the CTA's warps join: thread covers channels of a row in turn
  for (int i = threadIdx.x; i < kRows * DH; i += kThreads) {
    const int r = i / DH, d = i % DH;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][r]);
    float acc = 0.0f, ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = weight(s_m[w][r], M);
      acc = fmaf(f, s_o[(w * kRows + r) * DH + d], acc);
      ls = fmaf(f, s_l[w][r], ls);
    }
    s_o[r * DH + d] = acc;  // this element of warp 0's block is read by this thread alone
    if (d == 0) {
      s_cm[r] = M;
      s_cl[r] = ls;
    }
  }
  T* out = static_cast<T*>(p.out);
  auto store = [&](int r, int d, float v) {
    const int row = r0 + r;
    out[(static_cast<size_t>(b) * p.Sq + row / p.g) * p.ldo + (static_cast<size_t>(hkv) * p.g + row % p.g) * DH +
        d] = from_f<T>(v);
  };
  const int n_rows = last - r0 + 1;  // rows of this tile that exist
  if (p.C == 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * DH; i += kThreads) {
      const float L = s_cl[i / DH];
      store(i / DH, i % DH, L == 0.0f ? 0.0f : s_o[i] / L);
    }
    return;
  }
  cluster_sync_all();
  for (int i = rank * kThreads + threadIdx.x; i < n_rows * DH; i += p.C * kThreads) {
    const int r = i / DH;
    float M = -INFINITY;
    for (int c = 0; c < p.C; ++c) M = fmaxf(M, ld_dsmem(smem_u32(&s_cm[r]), c));
    float acc = 0.0f, L = 0.0f;
    for (int c = 0; c < p.C; ++c) {
      const float f = weight(ld_dsmem(smem_u32(&s_cm[r]), c), M);
      acc = fmaf(f, ld_dsmem(smem_u32(&s_o[i]), c), acc);
      L = fmaf(f, ld_dsmem(smem_u32(&s_cl[r]), c), L);
    }
    store(r, i % DH, L == 0.0f ? 0.0f : acc / L);
  }
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <typename T, int DH>
int launch(const AttnKvParams& p, unsigned tiles, cudaStream_t s) {
  constexpr int smem = kWarps * kRows * DH * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * p.C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  DLM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attn_kv_kernel<T, DH>, p));
  return DLM_OK;
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
  DLM_REQUIRE(scale > -INFINITY && scale < INFINITY, DLM_ERR_INVALID, "attention_kv_i8: scale is not finite");
  const int g = Hq / Hkv;
  const long long row_tiles = (static_cast<long long>(Sq) * g + kRows - 1) / kRows;
  const long long tiles = row_tiles * B * Hkv;
  DLM_REQUIRE(tiles < (1ll << 27) && static_cast<long long>(Sq) * g < (1ll << 30), DLM_ERR_UNSUPPORTED,
              "attention_kv_i8: too many rows");
  // CTAs per cluster: enough to fill the SMs twice, as long as each warp has keys to take
  int C = 1;
  while (C < 8 && tiles * C < 2ll * num_sms() && 2ll * C * kWarps * kUnit <= Lmax) C *= 2;
  AttnKvParams p{q, kq, kscale, vq, vscale, out, kv_len, q_len, ldq, ldo, B, Hq, Hkv, Sq, Lmax, g,
                 static_cast<int>(row_tiles), causal, C, scale * 1.4426950408889634f, device_status_ptr()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DLM_DISPATCH_DTYPE(dtype, T, {
    if (Dh == 64) return launch<T, 64>(p, static_cast<unsigned>(tiles), s);
    return launch<T, 128>(p, static_cast<unsigned>(tiles), s);
  });
}
