// Shared parts of the attention kernels with a relative position bias and / or key counts (attn_var*.hip).
//
// Scores are handled in units of 1 / scale:  S' = q k + T / scale,  p = exp2((S' - m) c),  c = scale log2 e.
// Row statistics kept for the backward pass: m (the reference maximum the exponentials were taken with) and lr = -log2 of
// their sum; a row that nothing is left for has m = 0, lr = -inf, so that every probability of it comes out 0.
#pragma once
#include "attn_share.h"
#include "attn_tile.h"

struct VarP {
  const void *q, *k, *v, *dout;
  void *o, *dq, *dk, *dv;
  float *stat, *delta;         // [B, H, Lq, 2] (m, lr); [B, H, Lq] rowsum(dO O), in the bf16 kernels with its sign turned
  float* nl;                   // [B, H, Lq] -m c + lr
  const int32_t* kv_len;
  const void* table;           // [buckets][H]
  const uint16_t* index;       // [Lq][Lk]
  const bf16 *bias_s, *bias_t; // the bias laid out in accumulator order (var_expand_k), keys or queries on the rows
  float* dbias;                // [splits][H][Lq][Lk]
  float* part;                 // split forward: [splits][B, H, Lq][Dh]; few-query backward: [blocks][B, H, Lq][Dh]
  float* pstat;                // split forward: [splits][B, H, Lq][2] (m, sum); few-query backward with a table's gradient:
                               // [blocks][B, H, Lq][2] (sum P dP, sum P), otherwise NULL
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss, v_sb, v_sh, v_ss, o_sb, o_sh, o_ss, g_sb, g_sh, g_ss;
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int B, H, Lq, Lk, Dh;
  int nqt, nkt;                // 32-row tiles of bias_s per head: nqt x nkt (nkt even); bias_t: nkt_t x nqt_t (nqt_t even)
  int nqt_t, nkt_t;
  int splits, buckets;
  uint64_t seed;
  float scale, inv_scale, bias_lim, keep_scale;
  uint32_t thr;
};

__device__ __forceinline__ int key_count(const VarP& p, int64_t b) {
  if (!p.kv_len) return p.Lk;
  // a scalar load: a vector load would be waited for together with every request in flight
  const int n = ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p.kv_len)[b];
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

// ---- streamed tiles: 64 rows x DHP bf16 values, brought into LDS by DMA -----------------------------------------------------
// A request moves 64 x 16 bytes to consecutive LDS addresses in lane order, so the rows are not padded; instead the source
// address is permuted: 16-byte chunk c of row r lies at position c ^ u_swz(r).  With it the row-wise 16-byte reads (16 rows at
// a time) and the transposing reads (4 rows x 64 bytes) of the fragments both spread over all banks.  Nothing passes through
// registers on the way, which is what lets these kernels hold their accumulators without spilling: a spilled register's
// reload waits behind every load in flight.  Rows at or beyond the descriptor's end arrive as zeros.
template <int DHP> __device__ __forceinline__ int u_swz(int row) {
  return DHP == 64 ? ((row >> 1) & 1) * 4 + ((row >> 2) & 3) : DHP == 96 ? (row >> 2) & 3 : (row & 3) * 4 + ((row >> 2) & 3);
}
template <int DHP> constexpr int u_tile() { return 64 * DHP * 2; }   // bytes
// element j = tile[r0 + (lane & 31)][ks*16 + 8*(lane >> 5) + j]   (r0 a multiple of 32)
template <int DHP> __device__ __forceinline__ bf16x8 u_rows(const char* s, int r0, int ks, int lane) {
  const int rl = lane & 31, hi = lane >> 5, f = u_swz<DHP>(rl);
  if (DHP == 96) return *(const bf16x8*)(s + rl * 192 + ((((ks & 1) * 2) | hi) ^ f) * 16 + (r0 * 192 + (ks >> 1) * 64));
  return *(const bf16x8*)(s + r0 * DHP * 2 + ((rl * DHP * 2 + (hi ^ f) * 16) ^ (ks * 32)));
}
// element j = tile[r0 + 16*s2 + 8*(j>>2) + 4*(lane>>5) + (j&3)][c0 + (lane&31)]   (r0, c0 multiples of 32): see frag_cols
template <int DHP> __device__ __forceinline__ bf16x8 u_cols(const char* s, int r0, int s2, int c0, int lane) {
  const int hi = lane >> 5, l3 = lane & 3;
  const int rowl = 4 * hi + ((lane & 15) >> 2), cl = 2 * ((lane >> 4) & 1) + (l3 >> 1), sub = (l3 & 1) * 8;
  const int f_lo = u_swz<DHP>(rowl), f_hi = u_swz<DHP>(rowl + 8);   // adding 16 to a row leaves u_swz as it is
  const char* t = s + (r0 + 16 * s2) * DHP * 2;
  int lo = rowl * DHP * 2 + (cl ^ f_lo) * 16 + sub, hi8 = (rowl + 8) * DHP * 2 + (cl ^ f_hi) * 16 + sub;
  if (DHP == 96) { lo += c0 * 2; hi8 += c0 * 2; }
  else { lo ^= c0 * 2; hi8 ^= c0 * 2; }
  const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(t + lo));
  const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(t + hi8));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
// The requests are issued from inline assembly: for a DMA it can see the compiler waits before every LDS read that follows.
// They write LDS, no register; u_wait / the barrier behind it order them against the reads.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is reserved; nothing else in these kernels uses it
__device__ __forceinline__ void u_dma16(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(uniform(lds)), "v"(voff), "s"(rs), "s"(uniform(soff)) : "memory", "m0");
}
__device__ __forceinline__ void u_dma4(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(uniform(lds)), "v"(voff), "s"(rs) : "memory", "m0");
}
#pragma clang diagnostic pop
// waits until at most N of the wave's memory requests are outstanding (they retire in the order of their issue)
template <int N> __device__ __forceinline__ void u_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(__attribute__((address_space(3))) const char*)p);
}
// One wave's share of a tile: DHP / 8 / NW requests
template <int DHP, int NW> struct TileDma {
  static constexpr int N = DHP / 8 / NW;
  __amdgpu_buffer_rsrc_t rs;
  uint32_t voff[N], tile_bytes, dst;
  int last;   // tile
};
template <int DHP, int NW>
__device__ __forceinline__ TileDma<DHP, NW> tile_dma(const bf16* g, int64_t ss, int S, int Dh, uint32_t dst, int wid, int lane) {
  constexpr int CPR = DHP / 8, N = CPR / NW;
  TileDma<DHP, NW> t;
  t.rs = rows_rsrc(g, ss, S, Dh);
  t.tile_bytes = (uint32_t)(64 * ss * 2);
  t.dst = dst + (uint32_t)(wid * N * 1024);
  t.last = (S - 1) >> 6;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int u = (wid * N + i) * 64 + lane, row = u / CPR, c = (u - row * CPR) ^ u_swz<DHP>(row);
    t.voff[i] = c * 8 < Dh ? (uint32_t)((row * ss + c * 8) * 2) : OOB_OFF;
  }
  return t;
}
// A tile beyond the last brings the last once more (no caller multiplies it): the scalar offset has to stay below the
// descriptor's size, which the hardware reduces by it before it compares.
template <int DHP, int NW> __device__ __forceinline__ void tile_request(const TileDma<DHP, NW>& t, int tile, uint32_t buf_off) {
  const uint32_t soff = (uint32_t)max(min(tile, t.last), 0) * t.tile_bytes;
#pragma unroll
  for (int i = 0; i < TileDma<DHP, NW>::N; i++) u_dma16(t.rs, t.voff[i], soff, t.dst + buf_off + i * 1024);
}

// The same for a wave of its own: 32 rows.  Its LDS reads have to be over (u_wait_lds) before their place is asked for again.
template <int DHP> struct WaveDma {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t voff[DHP / 16], tile_bytes, dst;
  int last;
};
template <int DHP> __device__ __forceinline__ WaveDma<DHP> wave_dma(const bf16* g, int64_t ss, int S, int Dh, uint32_t dst, int lane) {
  constexpr int CPR = DHP / 8;
  WaveDma<DHP> t;
  t.rs = rows_rsrc(g, ss, S, Dh);
  t.tile_bytes = (uint32_t)(32 * ss * 2);
  t.dst = dst;
  t.last = (S - 1) >> 5;
#pragma unroll
  for (int i = 0; i < DHP / 16; i++) {
    const int u = i * 64 + lane, row = u / CPR, c = (u - row * CPR) ^ u_swz<DHP>(row);
    t.voff[i] = c * 8 < Dh ? (uint32_t)((row * ss + c * 8) * 2) : OOB_OFF;
  }
  return t;
}
template <int DHP> __device__ __forceinline__ void wave_request(const WaveDma<DHP>& t, int tile, uint32_t buf_off) {
  const uint32_t soff = (uint32_t)max(min(tile, t.last), 0) * t.tile_bytes;
#pragma unroll
  for (int i = 0; i < DHP / 16; i++) u_dma16(t.rs, t.voff[i], soff, t.dst + buf_off + i * 1024);
}
__device__ __forceinline__ void u_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// launches of the matrix-unit kernels (attn_var_fwd.hip, attn_var_bwd.hip); operands checked by the caller
void var_launch_expand(const VarP& p, bool both, hipStream_t st);   // bias_s, or bias_s and bias_t
int var_few_heads(int64_t H);
void var_launch_few_fwd(const VarP& p, bool bias, hipStream_t st);
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
