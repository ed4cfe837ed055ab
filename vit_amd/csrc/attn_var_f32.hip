// float32 kernels on the matrix units (v_mfma_f32_32x32x2_f32) of attention with a relative position bias and / or key counts.
//
// The accumulator layout is that of the bf16 kernels (row index on the registers, column on the lane), and an operand of the
// 32x32x2 product is one value per lane: row or column = lane & 31, contraction index = lane >> 5.  Two consequences:
//   * the contraction over d may take its indices in any order, so the lane halves take 4 consecutive d each and one 16-byte
//     LDS read serves four products;
//   * the contraction over accumulator rows takes register r of both halves, rows acc_row(r) and acc_row(r) + 4: P and dS are
//     the next product's operand as they stand.
// An element of S costs 4 Dh operations at 256 per cycle and CU, a sixteenth of the bf16 rate, so everything else (exponentials,
// bias gathered from table and index where it is used, dropout) has room beside the matrix units.  Streamed tiles hold 32
// rows, in LDS, the next one on its way in registers.  ViT-S/16, 8 samples x 6 heads of 64, 197 x 197 with bias: forward 26 + 8,
// dQ 30, dK/dV 33, bias gradient 20 us (one wave per 32 rows without sharing: dQ 58, dK/dV 68); 4 x 12 heads, 77 queries over up
// to 577 states: 20 + 6, 27, 28 us (dQ 84 unshared).  At these sizes it is latency that counts, of the gathers, loads and products
// of one tile after the other: matrix units 10-16 % busy, vector instructions issued in 3-9 % of the cycles, 0.4-0.9 waves per SIMD.
#include "attn_var.h"

#define MFMA32 __builtin_amdgcn_mfma_f32_32x32x2f32

template <int DHP> struct F32Tile { static constexpr int STRIDE = DHP + 4, FLOATS = 32 * STRIDE; };

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc32(const float* g, int64_t ss, int S, int Dh) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)g, 0, S > 0 ? (int)(((int64_t)(S - 1) * ss + Dh) * 4) : 0, 0x00020000);
}
__device__ __forceinline__ f32x4 buf_load4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
// 32 rows x Dh from row0 on (rows at or beyond the descriptor's end and columns beyond Dh read as zeros)
template <int DHP, int NT, int NCH>
__device__ __forceinline__ void f32_load(f32x4 (&r)[NCH], __amdgpu_buffer_rsrc_t rs, int64_t ss, int row0, int Dh, int tid) {
  constexpr int CPR = DHP / 4;
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int c = tid + i * NT, row = c / CPR, d = (c % CPR) * 4;
    r[i] = buf_load4(rs, (c < 32 * CPR && d < Dh) ? (uint32_t)(((row0 + row) * ss + d) * 4) : OOB_OFF);
  }
}
template <int DHP, int NT, int NCH>
__device__ __forceinline__ void f32_store(const f32x4 (&r)[NCH], float* s, int tid) {
  constexpr int CPR = DHP / 4;
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int c = tid + i * NT, row = c / CPR, d = (c % CPR) * 4;
    if (c < 32 * CPR) *(f32x4*)(s + row * F32Tile<DHP>::STRIDE + d) = r[i];
  }
}
// operand with the row (or column) on the lane: group g holds d = 8 g + 4 (lane >> 5) + 0..3
template <int DHP>
__device__ __forceinline__ void f32_stationary(f32x4 (&f)[DHP / 8], const float* g, int64_t ss, int row, int S, int Dh, int lane) {
  const __amdgpu_buffer_rsrc_t rs = rows_rsrc32(g, ss, S, Dh);
#pragma unroll
  for (int i = 0; i < DHP / 8; i++) {
    const int d = 8 * i + 4 * (lane >> 5);
    f[i] = buf_load4(rs, (row < S && d < Dh) ? (uint32_t)((row * ss + d) * 4) : OOB_OFF);
  }
}
template <int DHP> __device__ __forceinline__ f32x4 f32_rows(const float* s, int g, int lane) {
  return *(const f32x4*)(s + (lane & 31) * F32Tile<DHP>::STRIDE + 8 * g + 4 * (lane >> 5));
}
// operand whose contraction index is the tile's row acc_row(r) + 4 (lane >> 5): column c0 + (lane & 31)
template <int DHP> __device__ __forceinline__ float f32_cols(const float* s, int r, int c0, int lane) {
  return s[(acc_row(r) + 4 * (lane >> 5)) * F32Tile<DHP>::STRIDE + c0 + (lane & 31)];
}
template <int DHP>
__device__ __forceinline__ void f32_product(f32x16& acc, const float* s, const f32x4 (&f)[DHP / 8], int lane) {
#pragma unroll
  for (int g = 0; g < DHP / 8; g++) {
    const f32x4 a = f32_rows<DHP>(s, g, lane);
#pragma unroll
    for (int j = 0; j < 4; j++) acc = MFMA32(a[j], f[g][j], acc, 0, 0, 0);
  }
}
template <int DHP>   // acc^T[d][lane] += tile^T[d][row] x[row][lane]
__device__ __forceinline__ void f32_accumulate(f32x16 (&acc)[DHP / 32], const float* s, const f32x16& x, int lane) {
#pragma unroll
  for (int r = 0; r < 16; r++)
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) acc[dt] = MFMA32(f32_cols<DHP>(s, r, dt * 32, lane), x[r], acc[dt], 0, 0, 0);
}
template <int DHP>
__device__ __forceinline__ void f32_store_rows(float* dst, const f32x16 (&acc)[DHP / 32], float mul, int Dh, int lane) {
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int d = dt * 32 + 8 * g + 4 * (lane >> 5);
      if (d < Dh) *(f32x4*)(dst + d) = f32x4{acc[dt][4 * g] * mul, acc[dt][4 * g + 1] * mul, acc[dt][4 * g + 2] * mul, acc[dt][4 * g + 3] * mul};
    }
}
// initial scores of a 32 x 32 tile: the bias of (query, key) in units of 1 / scale, 0 outside Lq x Lk.  KEYS_ON_ROWS: query on
// the lane.  All 16 buckets are asked for at once, then all 16 values.
template <bool KEYS_ON_ROWS>
__device__ __forceinline__ f32x16 f32_bias(const VarP& p, int h, int q0, int k0, int lane) {
  f32x16 a = ZERO16;
  if (p.table && q0 < p.Lq) {
    const __amdgpu_buffer_rsrc_t irs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.index + (int64_t)q0 * p.Lk), 0, min(32, p.Lq - q0) * p.Lk * 2, 0x00020000);
    const __amdgpu_buffer_rsrc_t trs = __builtin_amdgcn_make_buffer_rsrc((void*)((const float*)p.table + h), 0, (p.buckets * p.H - h) * 4, 0x00020000);
    const int base = (KEYS_ON_ROWS ? (lane & 31) * p.Lk + 4 * (lane >> 5) : 4 * (lane >> 5) * p.Lk + (lane & 31)) + k0;
    const int step = KEYS_ON_ROWS ? 1 : p.Lk, i0 = q0 + (KEYS_ON_ROWS ? (lane & 31) : 4 * (lane >> 5)), j0 = k0 + (KEYS_ON_ROWS ? 4 * (lane >> 5) : (lane & 31));
    uint32_t bucket[16];
#pragma unroll
    for (int r = 0; r < 16; r++) bucket[r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(irs, (base + acc_row(r) * step) * 2, 0, 0);
#pragma unroll
    for (int r = 0; r < 16; r++) a[r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(trs, (int)(bucket[r] * (uint32_t)p.H * 4u), 0, 0));
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const bool in = i0 + (KEYS_ON_ROWS ? 0 : acc_row(r)) < p.Lq && j0 + (KEYS_ON_ROWS ? acc_row(r) : 0) < p.Lk;
      a[r] = in ? clamp_bias(a[r], p.bias_lim) * p.inv_scale : 0.f;
    }
  }
  return a;
}

template <int DHP, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64) void f32_fwd_k(VarP p) {
  constexpr int NT = NW * 64, NCH = (32 * (DHP / 4) + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) float sK[F32Tile<DHP>::FLOATS], sV[F32Tile<DHP>::FLOATS];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = head_block(p.B, p.H, S, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int q0 = hb.xb * (NW * 32) + wid * 32, qrow = q0 + (lane & 31), rowoff = 4 * (lane >> 5);
  const bool wave_on = q0 < S;
  const KeyShare share = key_share(key_count(p, b), 32, SPLIT ? p.splits : 1, SPLIT ? (int)blockIdx.y : 0);
  const int t0 = share.t0, len = share.end, nt = share.t1;
  const __amdgpu_buffer_rsrc_t krs = rows_rsrc32((const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, len, Dh);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc32((const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, len, Dh);
  f32x4 qf[DHP / 8], rk[NCH], rv[NCH];
  f32_stationary<DHP>(qf, (const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qrow, S, Dh, lane);
  const f32x16 zero = ZERO16;
  f32x16 oacc[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) oacc[dt] = zero;
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;
  const uint32_t xrow = var_drop_xrow(p, (uint64_t)(b * p.H + h) * p.Lq + (uint64_t)qrow, lane);
  if (t0 < nt) {
    f32_load<DHP, NT, NCH>(rk, krs, p.k_ss, t0 * 32, Dh, tid);
    f32_load<DHP, NT, NCH>(rv, vrs, p.v_ss, t0 * 32, Dh, tid);
  }
  for (int t = t0; t < nt; t++) {
    __syncthreads();
    f32_store<DHP, NT, NCH>(rk, sK, tid);
    f32_store<DHP, NT, NCH>(rv, sV, tid);
    __syncthreads();
    f32_load<DHP, NT, NCH>(rk, krs, p.k_ss, (t + 1) * 32, Dh, tid);   // beyond the keys: zeros
    f32_load<DHP, NT, NCH>(rv, vrs, p.v_ss, (t + 1) * 32, Dh, tid);
    if (!wave_on) continue;
    f32x16 s = f32_bias<true>(p, (int)h, q0, t * 32, lane);
    f32_product<DHP>(s, sK, qf, lane);
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; r++) {
      if (t * 32 + acc_row(r) + rowoff >= len) s[r] = -INFINITY;
      mx = fmaxf(mx, s[r]);
    }
    mx = max_xor32(mx);
    const float mnew = fmaxf(m, mx), ms = mnew == -INFINITY ? 0.f : mnew;
    const float alpha = m == mnew ? 1.f : fast_exp2((m - mnew) * c);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[dt][r] *= alpha;
#pragma unroll
    for (int r = 0; r < 16; r++) { s[r] = fast_exp2((s[r] - ms) * c); l += s[r]; }
    if (p.thr) {
#pragma unroll
      for (int g = 0; g < 4; g++) {
        uint32_t dr[4];
        rng_lin_run<4>(xrow + (uint32_t)((t * 32 + acc_row(4 * g)) >> 1) * RNG_C1, dr);
#pragma unroll
        for (int j = 0; j < 4; j++) s[4 * g + j] = dr[j] < p.thr ? 0.f : s[4 * g + j] * p.keep_scale;
      }
    }
    f32_accumulate<DHP>(oacc, sV, s, lane);
  }
  l += __shfl_xor(l, 32, 64);
  if (qrow >= S) return;
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  if (SPLIT) {
    const int64_t prow = (int64_t)blockIdx.y * p.B * p.H * p.Lq + srow;
    f32_store_rows<DHP>(p.part + prow * Dh, oacc, 1.f, Dh, lane);
    if (lane < 32) { p.pstat[2 * prow] = m; p.pstat[2 * prow + 1] = l; }
    return;
  }
  f32_store_rows<DHP>((float*)p.o + b * p.o_sb + h * p.o_sh + (int64_t)qrow * p.o_ss, oacc, l == 0.f ? 0.f : 1.f / l, Dh, lane);
  if (lane < 32) {
    p.stat[2 * srow] = l == 0.f ? 0.f : m;
    p.stat[2 * srow + 1] = l == 0.f ? -INFINITY : -__log2f(l);
  }
}

// dS^T, in d, of a 32 x 32 tile with the keys k0 + acc_row on the registers and the query on the lane
template <bool DROP>
__device__ __forceinline__ void f32_dq_grads(const VarP& p, const f32x16& s, f32x16& d, float m, float lr, float delta, float c,
                                             uint32_t xrow, int k0, int len, int rowoff) {
#pragma unroll
  for (int g = 0; g < 4; g++) {
    uint32_t dr[4];
    if (DROP) rng_lin_run<4>(xrow + (uint32_t)((k0 + acc_row(4 * g)) >> 1) * RNG_C1, dr);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int r = 4 * g + j;
      float dp = d[r];
      if (DROP) dp = dr[j] < p.thr ? 0.f : dp * p.keep_scale;
      d[r] = k0 + acc_row(r) + rowoff < len ? fast_exp2((s[r] - m) * c + lr) * (dp - delta) : 0.f;
    }
  }
}

template <int DHP, int NW, bool DROP>
__global__ __launch_bounds__(NW * 64) void f32_dq_k(VarP p) {
  constexpr int NT = NW * 64, NCH = (32 * (DHP / 4) + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) float sK[F32Tile<DHP>::FLOATS], sV[F32Tile<DHP>::FLOATS];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = head_block(p.B, p.H, S, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int q0 = hb.xb * (NW * 32) + wid * 32, qrow = q0 + (lane & 31), rowoff = 4 * (lane >> 5);
  const bool wave_on = q0 < S, qv = qrow < S;
  const int len = key_count(p, b), nt = (len + 31) >> 5;
  const __amdgpu_buffer_rsrc_t krs = rows_rsrc32((const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, len, Dh);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc32((const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, len, Dh);
  f32x4 qf[DHP / 8], gf[DHP / 8], rk[NCH], rv[NCH];
  f32_stationary<DHP>(qf, (const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qrow, S, Dh, lane);
  f32_stationary<DHP>(gf, (const float*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, qrow, S, Dh, lane);
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  float delta = 0.f;
  {
    f32x4 of[DHP / 8];
    f32_stationary<DHP>(of, (const float*)p.o + b * p.o_sb + h * p.o_sh, p.o_ss, qrow, S, Dh, lane);
#pragma unroll
    for (int g = 0; g < DHP / 8; g++)
#pragma unroll
      for (int j = 0; j < 4; j++) delta = fmaf(of[g][j], gf[g][j], delta);
    delta += __shfl_xor(delta, 32, 64);
    if (qv && lane < 32) p.delta[srow] = delta;
  }
  const float m = qv ? p.stat[2 * srow] : 0.f, lr = qv ? p.stat[2 * srow + 1] : -INFINITY, c = p.scale * LOG2E;
  const uint32_t xrow = var_drop_xrow(p, (uint64_t)srow, lane);
  const f32x16 zero = ZERO16;
  f32x16 dq[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) dq[dt] = zero;
  f32_load<DHP, NT, NCH>(rk, krs, p.k_ss, 0, Dh, tid);
  f32_load<DHP, NT, NCH>(rv, vrs, p.v_ss, 0, Dh, tid);
  for (int t = 0; t < nt; t++) {
    __syncthreads();
    f32_store<DHP, NT, NCH>(rk, sK, tid);
    f32_store<DHP, NT, NCH>(rv, sV, tid);
    __syncthreads();
    f32_load<DHP, NT, NCH>(rk, krs, p.k_ss, (t + 1) * 32, Dh, tid);
    f32_load<DHP, NT, NCH>(rv, vrs, p.v_ss, (t + 1) * 32, Dh, tid);
    if (!wave_on) continue;
    f32x16 s = f32_bias<true>(p, (int)h, q0, t * 32, lane), d = zero;
    f32_product<DHP>(s, sK, qf, lane);
    f32_product<DHP>(d, sV, gf, lane);
    f32_dq_grads<DROP>(p, s, d, m, lr, delta, c, xrow, t * 32, len, rowoff);
    f32_accumulate<DHP>(dq, sK, d, lane);
  }
  if (qv) f32_store_rows<DHP>((float*)p.dq + b * p.dq_sb + h * p.dq_sh + (int64_t)qrow * p.dq_ss, dq, p.scale, Dh, lane);
}

// P and dS of a 32 x 32 tile with the queries q0 + acc_row on the registers and the key on the lane.  On return s holds the P
// that multiplies dO, d holds dS.
struct RowConst32 { float m[16], lr[16], delta[16]; };
template <bool DROP>
__device__ __forceinline__ void f32_row_grads(const VarP& p, f32x16& s, f32x16& d, const RowConst32& rc, float c, int64_t row0, int krow, int lane) {
  const int rowoff = 4 * (lane >> 5);
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const float pr = fast_exp2((s[r] - rc.m[r]) * c + rc.lr[r]);
    float dp = d[r], pd = pr;
    if (DROP) {
      const bool keep = rng_u32(p.seed, (uint64_t)(row0 + acc_row(r) + rowoff) * var_drop_ld(p) + (uint64_t)krow) >= p.thr;
      pd = keep ? pr * p.keep_scale : 0.f;
      dp = keep ? dp * p.keep_scale : 0.f;
    }
    s[r] = pd;
    d[r] = pr * (dp - rc.delta[r]);
  }
}
// sC = m, lr, delta [32] each
template <bool DROP>
__device__ __forceinline__ void f32_tile_grads(const VarP& p, f32x16& s, f32x16& d, const float* sC, float c, int64_t row0, int krow, int lane) {
  RowConst32 rc;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int q = acc_row(r) + 4 * (lane >> 5);
    rc.m[r] = sC[q];
    rc.lr[r] = sC[32 + q];
    rc.delta[r] = sC[64 + q];
  }
  f32_row_grads<DROP>(p, s, d, rc, c, row0, krow, lane);
}
__device__ __forceinline__ float f32_row_const(const VarP& p, int64_t sbase, int q0, int tid) {   // threads 0 .. 95
  const int which = tid >> 5, q = q0 + (tid & 31);
  if (q >= p.Lq) return which == 1 ? -INFINITY : 0.f;
  return which == 2 ? p.delta[sbase + q] : p.stat[2 * (sbase + q) + which];
}

template <int DHP, int NW, bool DROP>
__global__ __launch_bounds__(NW * 64) void f32_dkdv_k(VarP p) {
  constexpr int NT = NW * 64, NCH = (32 * (DHP / 4) + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) float sQ[F32Tile<DHP>::FLOATS], sG[F32Tile<DHP>::FLOATS], sC[96];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh;
  const HeadBlock hb = head_block(p.B, p.H, p.Lk, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int len = key_count(p, b), key0 = hb.xb * (NW * 32), k0 = key0 + wid * 32, krow = k0 + (lane & 31);
  const bool wave_on = k0 < len;
  const f32x16 zero = ZERO16;
  f32x16 dk[DHP / 32], dv[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; }
  if (key0 < len) {
    const __amdgpu_buffer_rsrc_t qrs = rows_rsrc32((const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, p.Lq, Dh);
    const __amdgpu_buffer_rsrc_t grs = rows_rsrc32((const float*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, p.Lq, Dh);
    f32x4 kf[DHP / 8], vf[DHP / 8], rq[NCH], rg[NCH];
    f32_stationary<DHP>(kf, (const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, krow, len, Dh, lane);
    f32_stationary<DHP>(vf, (const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, krow, len, Dh, lane);
    const int64_t sbase = (b * p.H + h) * p.Lq;
    const float c = p.scale * LOG2E;
    const int nt = (p.Lq + 31) >> 5;
    f32_load<DHP, NT, NCH>(rq, qrs, p.q_ss, 0, Dh, tid);
    f32_load<DHP, NT, NCH>(rg, grs, p.g_ss, 0, Dh, tid);
    for (int t = 0; t < nt; t++) {
      __syncthreads();
      f32_store<DHP, NT, NCH>(rq, sQ, tid);
      f32_store<DHP, NT, NCH>(rg, sG, tid);
      for (int i = tid; i < 96; i += NT) sC[i] = f32_row_const(p, sbase, t * 32, i);
      __syncthreads();
      f32_load<DHP, NT, NCH>(rq, qrs, p.q_ss, (t + 1) * 32, Dh, tid);
      f32_load<DHP, NT, NCH>(rg, grs, p.g_ss, (t + 1) * 32, Dh, tid);
      if (!wave_on) continue;
      f32x16 s = f32_bias<false>(p, (int)h, t * 32, k0, lane), d = zero;
      f32_product<DHP>(s, sQ, kf, lane);
      f32_product<DHP>(d, sG, vf, lane);
      f32_tile_grads<DROP>(p, s, d, sC, c, sbase + t * 32, krow, lane);
      f32_accumulate<DHP>(dv, sG, s, lane);
      f32_accumulate<DHP>(dk, sQ, d, lane);
    }
  }
  if (krow >= p.Lk) return;
  if (krow >= len) {   // padding: its columns hold whatever the zero rows gave
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; }
  }
  f32_store_rows<DHP>((float*)p.dv + b * p.dv_sb + h * p.dv_sh + (int64_t)krow * p.dv_ss, dv, 1.f, Dh, lane);
  f32_store_rows<DHP>((float*)p.dk + b * p.dk_sb + h * p.dk_sh + (int64_t)krow * p.dk_ss, dk, p.scale, Dh, lane);
}

// ---- few rows: the waves of a workgroup share 32 rows -------------------------------------------------------------------------
// Where 32 rows per wave leave most of the 1024 SIMDs idle (8 samples of ViT-S/16: 336 waves), the W waves of a workgroup take
// every W-th tile of the streamed rows for the same 32 stationary ones and add their sums up, in a fixed order, at the end.  A
// product of 32 x 32 x 2 takes 64 cycles, so the operands come straight from the caches: no
// staging in LDS, and no barrier until the end.
template <int DHP>   // rows row0 + (lane & 31), as f32_rows; rows at or beyond the descriptor's end and columns beyond Dh: zeros
__device__ __forceinline__ void f32_fetch_rows(f32x4 (&f)[DHP / 8], __amdgpu_buffer_rsrc_t rs, int64_t ss, int row0, int Dh, int lane) {
  const int d0 = 4 * (lane >> 5);
  const uint32_t off = (uint32_t)(((row0 + (lane & 31)) * (int)ss + d0) * 4);
#pragma unroll
  for (int i = 0; i < DHP / 8; i++) f[i] = buf_load4(rs, 8 * i + d0 < Dh ? off + 32u * i : OOB_OFF);
}
// as f32_cols; columns at or beyond Dh hold anything: they only reach result columns that are not stored
template <int DHP>
__device__ __forceinline__ void f32_fetch_cols(float (&f)[DHP / 32][16], __amdgpu_buffer_rsrc_t rs, int64_t ss, int row0, int lane) {
  const uint32_t off = (uint32_t)(((row0 + 4 * (lane >> 5)) * (int)ss + (lane & 31)) * 4);
#pragma unroll
  for (int r = 0; r < 16; r++)
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++)
      f[dt][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, (int)(off + (uint32_t)(acc_row(r) * (int)ss * 4) + 128u * dt), 0, 0));
}
template <int DHP>
__device__ __forceinline__ void f32_product2(f32x16& acc, const f32x4 (&a)[DHP / 8], const f32x4 (&f)[DHP / 8]) {
#pragma unroll
  for (int g = 0; g < DHP / 8; g++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc = MFMA32(a[g][j], f[g][j], acc, 0, 0, 0);
}
template <int DHP>
__device__ __forceinline__ void f32_accumulate2(f32x16 (&acc)[DHP / 32], const float (&f)[DHP / 32][16], const f32x16& x) {
#pragma unroll
  for (int r = 0; r < 16; r++)
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) acc[dt] = MFMA32(f[dt][r], x[r], acc[dt], 0, 0, 0);
}
// wave 0's acc += the other waves', pairwise: s holds DHP * 32 floats for half of the waves
template <int DHP> __device__ __forceinline__ void f32_join(f32x16 (&acc)[DHP / 32], float* s, int wid, int lane) {
  for (int n = (int)(blockDim.x >> 7); n > 0; n >>= 1) {
    __syncthreads();
    if (wid >= n && wid < 2 * n) {
      float* dst = s + (wid - n) * (DHP * 32) + lane;
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) dst[(dt * 16 + r) * 64] = acc[dt][r];
    }
    __syncthreads();
    if (wid < n) {
      const float* src = s + wid * (DHP * 32) + lane;
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[dt][r] += src[(dt * 16 + r) * 64];
    }
  }
}
template <int DHP> constexpr int f32_share_max() { return DHP <= 64 ? 8 : 4; }   // waves; the larger heads need a SIMD's registers
template <int DHP, bool DROP>
__global__ __launch_bounds__(f32_share_max<DHP>() * 64) void f32_dq_share_k(VarP p) {
  __shared__ float sJoin[f32_share_max<DHP>() / 2 * DHP * 32];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = (int)(blockDim.x >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = head_block(p.B, p.H, S, 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int q0 = hb.xb * 32, qrow = q0 + (lane & 31), rowoff = 4 * (lane >> 5);
  const bool qv = qrow < S;
  const int len = key_count(p, b), nt = (len + 31) >> 5;
  const __amdgpu_buffer_rsrc_t krs = rows_rsrc32((const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, len, Dh);
  const __amdgpu_buffer_rsrc_t vrs = rows_rsrc32((const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, len, Dh);
  f32x4 qf[DHP / 8], gf[DHP / 8];
  f32_stationary<DHP>(qf, (const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qrow, S, Dh, lane);
  f32_stationary<DHP>(gf, (const float*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, qrow, S, Dh, lane);
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  float delta = 0.f;
  {
    f32x4 of[DHP / 8];
    f32_stationary<DHP>(of, (const float*)p.o + b * p.o_sb + h * p.o_sh, p.o_ss, qrow, S, Dh, lane);
#pragma unroll
    for (int g = 0; g < DHP / 8; g++)
#pragma unroll
      for (int j = 0; j < 4; j++) delta = fmaf(of[g][j], gf[g][j], delta);
    delta += __shfl_xor(delta, 32, 64);
    if (qv && wid == 0 && lane < 32) p.delta[srow] = delta;
  }
  const float m = qv ? p.stat[2 * srow] : 0.f, lr = qv ? p.stat[2 * srow + 1] : -INFINITY, c = p.scale * LOG2E;
  const uint32_t xrow = var_drop_xrow(p, (uint64_t)srow, lane);
  const f32x16 zero = ZERO16;
  f32x16 dq[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) dq[dt] = zero;
  for (int t = wid; t < nt; t += W) {
    float kc[DHP / 32][16];
    f32x4 kf[DHP / 8], vf[DHP / 8];
    f32_fetch_rows<DHP>(kf, krs, p.k_ss, t * 32, Dh, lane);
    f32x16 s = f32_bias<true>(p, (int)h, q0, t * 32, lane), d = zero;
    f32_fetch_rows<DHP>(vf, vrs, p.v_ss, t * 32, Dh, lane);
    f32_product2<DHP>(s, kf, qf);
    f32_fetch_cols<DHP>(kc, krs, p.k_ss, t * 32, lane);
    f32_product2<DHP>(d, vf, gf);
    f32_dq_grads<DROP>(p, s, d, m, lr, delta, c, xrow, t * 32, len, rowoff);
    f32_accumulate2<DHP>(dq, kc, d);
  }
  f32_join<DHP>(dq, sJoin, wid, lane);
  if (qv && wid == 0) f32_store_rows<DHP>((float*)p.dq + b * p.dq_sb + h * p.dq_sh + (int64_t)qrow * p.dq_ss, dq, p.scale, Dh, lane);
}
template <int DHP, bool DROP>
__global__ __launch_bounds__(f32_share_max<DHP>() * 64) void f32_dkdv_share_k(VarP p) {
  __shared__ float sJoin[f32_share_max<DHP>() / 2 * DHP * 32];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = (int)(blockDim.x >> 6), Dh = p.Dh;
  const HeadBlock hb = head_block(p.B, p.H, p.Lk, 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int len = key_count(p, b), k0 = hb.xb * 32, krow = k0 + (lane & 31);
  const f32x16 zero = ZERO16;
  f32x16 dk[DHP / 32], dv[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; }
  if (k0 < len) {
    const __amdgpu_buffer_rsrc_t qrs = rows_rsrc32((const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, p.Lq, Dh);
    const __amdgpu_buffer_rsrc_t grs = rows_rsrc32((const float*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, p.Lq, Dh);
    f32x4 kf[DHP / 8], vf[DHP / 8];
    f32_stationary<DHP>(kf, (const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, krow, len, Dh, lane);
    f32_stationary<DHP>(vf, (const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, krow, len, Dh, lane);
    const int64_t sbase = (b * p.H + h) * p.Lq;
    const float c = p.scale * LOG2E;
    const int nt = (p.Lq + 31) >> 5;
    for (int t = wid; t < nt; t += W) {
      float fc[DHP / 32][16];
      f32x4 qf[DHP / 8], gf[DHP / 8];
      const int qrow = t * 32 + (lane & 31);
      const bool in = qrow < p.Lq;   // others: zeros, as their Q and dO
      const float m = in ? p.stat[2 * (sbase + qrow)] : 0.f, lr = in ? p.stat[2 * (sbase + qrow) + 1] : 0.f, delta = in ? p.delta[sbase + qrow] : 0.f;
      f32_fetch_rows<DHP>(qf, qrs, p.q_ss, t * 32, Dh, lane);
      f32x16 s = f32_bias<false>(p, (int)h, t * 32, k0, lane), d = zero;
      f32_fetch_rows<DHP>(gf, grs, p.g_ss, t * 32, Dh, lane);
      f32_product2<DHP>(s, qf, kf);
      f32_product2<DHP>(d, gf, vf);
      __builtin_amdgcn_sched_barrier(0);   // the constants and the next operands are not to be live beside Q's and dO's rows
      RowConst32 rc;   // from the lane that holds the row's
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int at = acc_row(r) + 4 * (lane >> 5);
        rc.m[r] = __shfl(m, at, 64);
        rc.lr[r] = __shfl(lr, at, 64);
        rc.delta[r] = __shfl(delta, at, 64);
      }
      f32_fetch_cols<DHP>(fc, grs, p.g_ss, t * 32, lane);
      f32_row_grads<DROP>(p, s, d, rc, c, sbase + t * 32, krow, lane);
      f32_accumulate2<DHP>(dv, fc, s);
      f32_fetch_cols<DHP>(fc, qrs, p.q_ss, t * 32, lane);
      f32_accumulate2<DHP>(dk, fc, d);
    }
    f32_join<DHP>(dv, sJoin, wid, lane);
    f32_join<DHP>(dk, sJoin, wid, lane);
  }
  if (wid || krow >= p.Lk) return;
  if (krow >= len) {   // padding: its columns hold whatever the zero rows gave
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; }
  }
  f32_store_rows<DHP>((float*)p.dv + b * p.dv_sb + h * p.dv_sh + (int64_t)krow * p.dv_ss, dv, 1.f, Dh, lane);
  f32_store_rows<DHP>((float*)p.dk + b * p.dk_sb + h * p.dk_sh + (int64_t)krow * p.dk_ss, dk, p.scale, Dh, lane);
}

// dS summed over the samples of a share (gridDim.y shares): 32 queries x 128 keys per workgroup, 32 keys per wave
template <int DHP, bool DROP>
__global__ __launch_bounds__(256) void f32_dbias_k(VarP p) {
  constexpr int NT = 256, NCH = (32 * (DHP / 4) + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) float sQ[F32Tile<DHP>::FLOATS], sG[F32Tile<DHP>::FLOATS], sC[96];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh;
  const int nkb = (p.Lk + 127) / 128, nqb = (p.Lq + 31) / 32;
  const int kb = (int)blockIdx.x % nkb, rest = (int)blockIdx.x / nkb, qb = rest % nqb, h = rest / nqb;
  const int key0 = kb * 128, k0 = key0 + wid * 32, krow = k0 + (lane & 31), q0 = qb * 32;
  const int share = (p.B + (int)gridDim.y - 1) / (int)gridDim.y, b_end = min(p.B, share * ((int)blockIdx.y + 1));
  const f32x16 zero = ZERO16, bias = f32_bias<false>(p, h, q0, k0, lane);
  const float c = p.scale * LOG2E;
  f32x16 acc = zero;
  for (int b = share * (int)blockIdx.y; b < b_end; b++) {
    const int len = key_count(p, b);
    if (len <= key0) continue;
    const __amdgpu_buffer_rsrc_t qrs = rows_rsrc32((const float*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, p.Lq, Dh);
    const __amdgpu_buffer_rsrc_t grs = rows_rsrc32((const float*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, p.Lq, Dh);
    f32x4 kf[DHP / 8], vf[DHP / 8], rq[NCH], rg[NCH];
    f32_load<DHP, NT, NCH>(rq, qrs, p.q_ss, q0, Dh, tid);
    f32_load<DHP, NT, NCH>(rg, grs, p.g_ss, q0, Dh, tid);
    f32_stationary<DHP>(kf, (const float*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, krow, len, Dh, lane);
    f32_stationary<DHP>(vf, (const float*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, krow, len, Dh, lane);
    const int64_t sbase = ((int64_t)b * p.H + h) * p.Lq;
    __syncthreads();
    f32_store<DHP, NT, NCH>(rq, sQ, tid);
    f32_store<DHP, NT, NCH>(rg, sG, tid);
    if (tid < 96) sC[tid] = f32_row_const(p, sbase, q0, tid);
    __syncthreads();
    if (k0 >= len) continue;
    f32x16 s = bias, d = zero;
    f32_product<DHP>(s, sQ, kf, lane);
    f32_product<DHP>(d, sG, vf, lane);
    f32_tile_grads<DROP>(p, s, d, sC, c, sbase + q0, krow, lane);
    const bool live = krow < len;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] += live ? d[r] : 0.f;
  }
  if (krow >= p.Lk) return;
  float* out = p.dbias + ((int64_t)blockIdx.y * p.H + h) * p.Lq * p.Lk + krow;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int row = q0 + acc_row(r) + 4 * (lane >> 5);
    if (row < p.Lq) out[(int64_t)row * p.Lk] = acc[r];
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
#define F32_DH(...) do { if (p.Dh <= 32) { constexpr int D = 32; __VA_ARGS__; } else if (p.Dh <= 64) { constexpr int D = 64; __VA_ARGS__; } \
    else if (p.Dh <= 96) { constexpr int D = 96; __VA_ARGS__; } else { constexpr int D = 128; __VA_ARGS__; } } while (0)
// waves per workgroup (32 stationary rows each): 4 where that gives the chip enough workgroups, else 1
static int f32_nw(const VarP& p, int rows) { return (int64_t)p.B * p.H * ceil_div(rows, 128) >= 512 ? 4 : 1; }
// waves that share 32 of `rows`: as many as can run at once (two per SIMD, 2048 in all) and have a tile of the other rows
template <int DHP> static int f32_share(const VarP& p, int rows, int other) {
  const int64_t waves = (int64_t)p.B * p.H * ceil_div(rows, 32), tiles = ceil_div(other, 32);
  int w = 1;
  while (w < f32_share_max<DHP>() && 2 * w * waves <= 2048 && w < tiles) w *= 2;
  return w;
}
void f32_launch_fwd(const VarP& p, hipStream_t st) {
  F32_DH(
    if (p.splits > 1) hipLaunchKernelGGL((f32_fwd_k<D, 1, true>), dim3(head_block_grid(p.B, p.H, p.Lq, 32), p.splits), dim3(64), 0, st, p);
    else if (f32_nw(p, p.Lq) == 4) hipLaunchKernelGGL((f32_fwd_k<D, 4, false>), dim3(head_block_grid(p.B, p.H, p.Lq, 128)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((f32_fwd_k<D, 1, false>), dim3(head_block_grid(p.B, p.H, p.Lq, 32)), dim3(64), 0, st, p));
}
template <bool DROP> static void f32_bwd(const VarP& p, hipStream_t st) {
  F32_DH(
    if (f32_nw(p, p.Lq) == 4) hipLaunchKernelGGL((f32_dq_k<D, 4, DROP>), dim3(head_block_grid(p.B, p.H, p.Lq, 128)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((f32_dq_share_k<D, DROP>), dim3(head_block_grid(p.B, p.H, p.Lq, 32)), dim3(64 * f32_share<D>(p, p.Lq, p.Lk)), 0, st, p);
    if (f32_nw(p, p.Lk) == 4) hipLaunchKernelGGL((f32_dkdv_k<D, 4, DROP>), dim3(head_block_grid(p.B, p.H, p.Lk, 128)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((f32_dkdv_share_k<D, DROP>), dim3(head_block_grid(p.B, p.H, p.Lk, 32)), dim3(64 * f32_share<D>(p, p.Lk, p.Lq)), 0, st, p));
}
void f32_launch_bwd(const VarP& p, hipStream_t st) { if (p.thr) f32_bwd<true>(p, st); else f32_bwd<false>(p, st); }
void f32_launch_dbias(const VarP& p, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div(p.Lk, 128) * ceil_div(p.Lq, 32) * p.H), (unsigned)p.splits);
  if (p.thr) F32_DH(hipLaunchKernelGGL((f32_dbias_k<D, true>), grid, dim3(256), 0, st, p));
  else F32_DH(hipLaunchKernelGGL((f32_dbias_k<D, false>), grid, dim3(256), 0, st, p));
}
