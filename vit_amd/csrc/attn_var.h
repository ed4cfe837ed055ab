// Shared parts of the attention kernels with a relative position bias and / or key counts (attn_var*.hip).
//
// Scores are handled in units of 1 / scale:  S' = q k + T / scale,  p = exp2((S' - m) c),  c = scale log2 e.
// Row statistics kept for the backward pass: m (the reference maximum the exponentials were taken with) and lr = -log2 of
// their sum; a row that nothing is left for has m = 0, lr = -inf, so that every probability of it comes out 0.
#pragma once
#include "attn_tile.h"

struct VarP {
  const void *q, *k, *v, *dout;
  void *o, *dq, *dk, *dv;
  float *stat, *delta;         // [B, H, Lq, 2] (m, lr); [B, H, Lq] rowsum(dO O)
  const int32_t* kv_len;
  const void* table;           // [buckets][H]
  const uint16_t* index;       // [Lq][Lk]
  const bf16 *bias_s, *bias_t; // the bias laid out in accumulator order (var_expand_k), keys or queries on the rows
  float* dbias;                // [splits][H][Lq][Lk]
  float* part;                 // split forward: [splits][B, H, Lq][Dh]; few-query backward: [blocks][B, H, Lq][Dh]
  float* pstat;                // split forward: [splits][B, H, Lq][2] (m, sum)
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss, o_sb, o_sh, o_ss, g_sb, g_sh, g_ss;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int B, H, Lq, Lk, Dh;
  int nqt, nkt;                // 32-row tiles of bias_s per head: nqt x nkt (nkt even); bias_t: nkt_t x nqt_t (nqt_t even)
  int nqt_t, nkt_t;
  int splits;
  uint64_t seed;
  float scale, inv_scale, bias_lim, keep_scale;
  uint32_t thr;
};

__device__ __forceinline__ int key_count(const VarP& p, int64_t b) {
  if (!p.kv_len) return p.Lk;
  const int n = p.kv_len[b];
  return n < 0 ? 0 : n > p.Lk ? p.Lk : n;
}
// Finite entries beyond the limit are pulled in so that S' and its multiples stay finite; -inf, +inf and NaN pass.
__device__ __forceinline__ float clamp_bias(float x, float lim) {
  const float a = fabsf(x);
  return a > lim && a < INFINITY ? copysignf(lim, x) : x;
}
// dropout counter of (row, key): as in attn.hip, row * (Lk rounded up to even) + key
__device__ __forceinline__ uint64_t var_drop_ld(const VarP& p) { return (uint64_t)((p.Lk + 1) & ~1); }
__device__ __forceinline__ uint32_t var_drop_xrow(const VarP& p, uint64_t row, int lane) {
  return (uint32_t)(row * (var_drop_ld(p) >> 1)) * RNG_C1 + (uint32_t)(2 * (lane >> 5)) * RNG_C1 + rng_seedmix(p.seed);
}
// Exponents beyond this are not formed as fma(S', c, -m c): the rounding of the product m c would show (a row that holds
// nothing but a mask's lowest value); such tiles take (S' - m) c instead.
constexpr float BIG_EXP = 16384.f;

// Workgroup -> item for launches whose neighbouring items share data: workgroups go to the 8 XCDs round-robin and every XCD
// has an L2 of its own, so each XCD takes a contiguous eighth of the items.  Launched with xcd_grid(items) workgroups.
__device__ __forceinline__ int64_t xcd_item(int64_t L, int64_t items) {
  const int64_t n = (items + 7) >> 3, i = L >> 3, item = (L & 7) * n + i;
  return i < n && item < items ? item : -1;
}
static inline unsigned xcd_grid(int64_t items) { return (unsigned)(8 * ((items + 7) >> 3)); }
// Workgroup -> (sample, head, block of stationary rows).  With a bias the samples are neighbours: they read the same bias
// tiles, which are then fetched once per XCD and not once per sample (ViT-g/14 at 1024 px, 4 samples: 3.6 GB of bias per
// pass otherwise).  Without one the row blocks of a (sample, head) are: they share its streamed operands (head_block).
template <bool BIAS>
__device__ __forceinline__ HeadBlock var_block(const VarP& p, int nrows, int rows_per_block) {
  if (!BIAS) return head_block(p.B, p.H, nrows, rows_per_block);
  const int nxb = (nrows + rows_per_block - 1) / rows_per_block;
  const int64_t it = xcd_item(blockIdx.x, (int64_t)p.H * nxb * p.B);
  HeadBlock o;
  o.valid = it >= 0;
  const int64_t g = it / p.B;
  o.b = it - g * p.B;
  o.h = g / nxb;
  o.xb = (int)(g - o.h * nxb);
  return o;
}
template <bool BIAS> static inline unsigned var_grid(const VarP& p, int nrows, int rows_per_block) {
  if (!BIAS) return head_block_grid(p.B, p.H, nrows, rows_per_block);
  return xcd_grid((int64_t)p.H * ceil_div(nrows, rows_per_block) * p.B);
}

// launches of the matrix-unit kernels (attn_var_fwd.hip, attn_var_bwd.hip); operands checked by the caller
void var_launch_expand(const VarP& p, bool transposed, hipStream_t st);
void var_launch_fwd(const VarP& p, bool bias, int nw, hipStream_t st);
void var_launch_dq(const VarP& p, bool bias, hipStream_t st);
void var_launch_dkdv(const VarP& p, bool bias, hipStream_t st);
void var_launch_dbias(const VarP& p, hipStream_t st);
void var_launch_few_bwd(const VarP& p, bool bias, hipStream_t st);
void var_launch_combine(const VarP& p, bool f32, hipStream_t st);
// float32 (attn_var_f32.hip)
void f32_launch_fwd(const VarP& p, hipStream_t st);
void f32_launch_bwd(const VarP& p, hipStream_t st);
void f32_launch_dbias(const VarP& p, hipStream_t st);
