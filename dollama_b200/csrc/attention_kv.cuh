// Shared by the two kernels of attention over the int8 K/V cache (attention_kv.cu for a few rows per
// kv head, attention_kv_tc.cu for many).
#pragma once

#include <cstdint>

#include "dtype.cuh"
#include "ptx.cuh"

namespace dlm {

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
  int B, Hq, Hkv, Sq, Lmax;
  int g;          // query heads of a kv head
  int row_tiles;  // tiles of the rows (query, head of the group) of one (sequence, kv head)
  int tiles;      // of all of them
  int causal;
  int C;          // CTAs of a cluster, which share one tile's keys
  float scale_log2;
  int* status;
  int* bad_position;  // device status word of lengths outside the cache
};

// Rows (queries times heads of a group) above which the tensor-memory kernel runs: as many as the
// few-row kernel holds in registers.  Its tile of 64 keys costs about the same for 17 rows as for 128.
// 4 sequences, 8 kv heads, 16384 keys, fp16, us (cache bytes alone 11 / 21 for Dh 64 / 128):
//   rows                                       16         24         32         64        128
//   few-row kernel, a tile for every 16   23 / 35    35 / 56    36 / 56   59 / 100  124 / 177
//   tensor-memory kernel                              71 / 97    71 / 98    72 / 99   74 / 102
// and with 16 sequences of 512 keys 11 / 16 against 14 / 18 for 24 rows, 20 / 29 against 14 / 19 for
// 128: with long caches the border would lie nearer to 64 rows, with short ones at 32.
constexpr int kAttnKvFewRows = 16;

template <typename T, int DH>
int attn_kv_tc(const AttnKvParams& p, cudaStream_t s);

// One (sequence, kv head, row tile): its rows r0 .. last (row r: query r / g, head r % g) and the keys
// they see.  A length outside the cache is clamped and raises the device status word of positions.
struct AttnKvTile {
  int b, hkv, r0, last, n_kv, n_q, n_keys, n_all;

  __device__ __forceinline__ AttnKvTile(const AttnKvParams& p, int t, int rows_per_tile, bool report) {
    const int rt = t % p.row_tiles;
    t /= p.row_tiles;
    hkv = t % p.Hkv;
    b = t / p.Hkv;
    n_kv = p.kv_len[b];
    if (n_kv < 0 || n_kv > p.Lmax) {
      if (report && p.bad_position) *p.bad_position = kDevBadPosition;
      n_kv = n_kv < 0 ? 0 : p.Lmax;
    }
    n_q = p.q_len ? p.q_len[b] : p.Sq;
    n_q = n_q < 0 ? 0 : (n_q > p.Sq ? p.Sq : n_q);
    r0 = rt * rows_per_tile;
    const int rows = n_q * p.g;
    last = (r0 + rows_per_tile < rows ? r0 + rows_per_tile : rows) - 1;
    n_keys = last < r0 ? 0 : seen(p, last);  // the last row sees the most
    n_all = last < r0 ? 0 : seen(p, r0);     // keys that every row sees
  }
  // keys of row r: [0, seen)
  __device__ __forceinline__ int seen(const AttnKvParams& p, int r) const {
    if (!p.causal) return n_kv;
    const int e = n_kv - n_q + r / p.g + 1;
    return e < 0 ? 0 : e;
  }
  __device__ __forceinline__ size_t head(const AttnKvParams& p) const {
    return static_cast<size_t>(b) * p.Hkv + hkv;
  }
  template <typename T>
  __device__ __forceinline__ const T* q_row(const AttnKvParams& p, int r, int dh) const {
    return static_cast<const T*>(p.q) + (static_cast<size_t>(b) * p.Sq + r / p.g) * p.ldq +
           (static_cast<size_t>(hkv) * p.g + r % p.g) * dh;
  }
  template <typename T>
  __device__ __forceinline__ T* out_row(const AttnKvParams& p, int r, int dh) const {
    return static_cast<T*>(p.out) + (static_cast<size_t>(b) * p.Sq + r / p.g) * p.ldo +
           (static_cast<size_t>(hkv) * p.g + r % p.g) * dh;
  }
};

// The running reference of a row's weights: p_j = 2^(s_j - ref) and w_j = p_j vscale_j, with ref such
// that the largest |w| when ref was set is 2^kTarget and p stays below 2^100; ref starts at kNoRef and
// moves only when a weight would reach kMaxWeight or the sum kMaxSum.  Sum and products share the
// scale 2^-ref, so out = o / l.  A lower target makes moves rarer (each costs a second pass over the
// keys at hand: with 2^14 a tile of 128 keys x 32 rows moved one row or more most of the time, and
// 2x500 queries over 4096 keys took 150 us) and costs range: fp16 keeps 11 bits of a weight down to
// 2^-14, and an absolute 2^-25 below, which is 2^-35 of the largest weight for 16-bit types (2^-37 for
// fp32, whose second terms reach 22 bits down to 2^-15 of it).
constexpr float kNoRef = -1e30f, kMaxWeight = 60000.0f, kMaxSum = 0x1p122f;
template <typename T>
constexpr float kTarget = sizeof(T) == 4 ? 12.0f : 10.0f;
// A new reference from the largest score and the largest score + log2 |vscale| (-inf for none).
template <typename T>
__device__ __forceinline__ float new_ref(float ref, float top, float top_w) {
  return fmaxf(ref, fmaxf(top_w - kTarget<T>, top - 100.0f));
}
// score + log2 |vscale|, -inf where vscale is zero or not finite
__device__ __forceinline__ float weight_log2(float x, float vs) {
  const float a = fabsf(vs);
  return a > 0.0f && a < INFINITY ? x + __log2f(a) : -INFINITY;
}

// two biased codes (code + 128) picked by sel -> fp16 pair of the codes
__device__ __forceinline__ uint32_t code_pair(uint32_t biased, uint32_t sel) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, sel);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1152.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^e as a float for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }
// smallest e with |x| < 2^e for a normal x (the biased exponent alone)
__device__ __forceinline__ int exp_above(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 0xFF) - 126; }
// the exponent that scales a q row of largest magnitude mx to [2^14, 2^15) (rows below 2^-85 score 0)
__device__ __forceinline__ int q_up(float mx) { return min(15 - exp_above(mx), 100); }

// fp16 pair of two floats, and of what it leaves
__device__ __forceinline__ uint32_t half_pair(float a, float b) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t half_rest(uint32_t hi, float a, float b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return pack_half2(a - f.x, b - f.y);
}

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

// A launch of `grid` CTAs in clusters of C, with programmatic dependent launch.
template <typename P>
cudaError_t launch_clusters(void (*kernel)(P), unsigned grid, int threads, size_t smem, int C, cudaStream_t s,
                            const P& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace dlm
