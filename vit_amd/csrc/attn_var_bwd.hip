// Backward pass on the matrix units of attention with a relative position bias and / or key counts.
//
//   var_dq_k    queries stationary (32 per wave), K and V stream: S'^T and dP^T with the query on the lane, dQ^T += K^T dS^T
//   var_dkdv_k  keys stationary, Q and dO stream: S' and dP with the key on the lane, dV^T += dO^T P, dK^T += Q^T dS
//   var_dbias_k pairs stationary (128 x 64 per workgroup), samples stream: dS summed over the samples in the accumulators, in
//               32 bits, one 32-bit value per pair and head out; no atomics, so the sums do not depend on the order of anything
//   var_few_bwd_k up to 32 queries: keys stationary, everything in one pass over K and V (below)
// Times: ViT-B/14, 64 samples x 12 heads of 64, 272 x 272 with bias: dQ 62, dK/dV 71, bias gradient 60 us; ViT-g/14 at 1024 px, 4 x
// 16 heads of 88, 5329 x 5329 with bias: 1.25, 1.51, 2.10 ms; 300 queries over up to 4096 states, 16 x 16 heads of 64: dQ and
// dK/dV 280 us together (126 and 181 with a profiler attached).  All are bound by the latency of a wave's chain through a tile,
// which two or three waves per SIMD do not cover: matrix units 15-45 % busy (bias gradient 11-15), vector instructions issued in
// 29-44 % of the cycles (18-23), waves waiting 31-47 % of their time, LDS bank conflicts next to none.
// P is formed again from the row statistics of the forward pass; delta = rowsum(dO O) comes from var_dq_k / var_few_bwd_k.
#include "attn_var.h"

template <bool BIAS>
__device__ __forceinline__ f32x16 init_tile(const bf16x8& lo, const bf16x8& hi, float inv_scale) {
  f32x16 a = ZERO16;
  if (BIAS) {
#pragma unroll
    for (int r = 0; r < 8; r++) { a[r] = (float)lo[r] * inv_scale; a[8 + r] = (float)hi[r] * inv_scale; }
  }
  return a;
}

// ---- dQ -----------------------------------------------------------------------------------------------------------------
// WHOLE: the tile holds all keys of the rows, and delta = sum P dP / sum P replaces rowsum(dO O), whose rounding is much of what
// dS is made of when the keys are few (5 keys: error of dq 3.0e-3, 2.4e-3 so).
template <int DHP, int HALVES, bool PARTIAL, bool BIAS, bool DROP, bool WHOLE = false>
__device__ __forceinline__ void var_dq_tile(const VarP& p, const char* sK, const char* sV, const bf16x8 (&qf)[DHP / 16],
                                            const bf16x8 (&gf)[DHP / 16], f32x16 (&sacc)[HALVES], f32x16 (&dqacc)[DHP / 32],
                                            float m, float nmc, bool big, float& delta, float& dsum, float c, int k0, int len,
                                            uint32_t xrow, int lane) {
  const f32x16 zero = ZERO16;
  const int rowoff = 4 * (lane >> 5);
  auto scores = [&](int st, f32x16& pacc) {   // P in sacc, dP (dropout applied) in pacc
#pragma unroll
    for (int ks = 0; ks < DHP / 16; ks++) {
      sacc[st] = MFMA(u_rows<DHP>(sK, st * 32, ks, lane), qf[ks], sacc[st], 0, 0, 0);
      pacc = MFMA(u_rows<DHP>(sV, st * 32, ks, lane), gf[ks], pacc, 0, 0, 0);
    }
    if (BIAS && big) {
#pragma unroll
      for (int r = 0; r < 16; r++) sacc[st][r] = fast_exp2((sacc[st][r] - m) * c);
    } else {
#pragma unroll
      for (int r = 0; r < 16; r++) sacc[st][r] = fast_exp2(fmaf(sacc[st][r], c, nmc));
    }
#pragma unroll
    for (int g = 0; g < 4; g++) {   // registers 4 g .. 4 g + 3: four consecutive keys from a multiple of 4
      uint32_t dr[4] = {0u, 0u, 0u, 0u};
      if (DROP) rng_lin_run<4>(xrow + (uint32_t)((k0 + st * 32 + acc_row(4 * g)) >> 1) * RNG_C1, dr);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = 4 * g + j;
        if (PARTIAL && st == HALVES - 1) sacc[st][r] = k0 + st * 32 + acc_row(r) + rowoff < len ? sacc[st][r] : 0.f;
        if (DROP) pacc[r] = dr[j] >= p.thr ? pacc[r] * p.keep_scale : 0.f;
      }
    }
  };
  auto grads = [&](int st, const f32x16& pacc) {
#pragma unroll
    for (int r = 0; r < 16; r++) sacc[st][r] *= pacc[r] - delta;
    // dS is rounded to bf16 to be an operand (half a step, 2^-8); its row factor 1 / sum is applied to the 32-bit result
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      const bf16x8 df = acc_to_frag(sacc[st], s2);
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++)
        dqacc[dt] = MFMA(u_cols<DHP>(sK, st * 32, s2, dt * 32, lane), df, dqacc[dt], 0, 0, 0);
      if (BIAS && !WHOLE) {
#pragma unroll
        for (int r = 8 * s2; r < 8 * s2 + 8; r += 2) dsum += sacc[st][r] + sacc[st][r + 1];
      }
    }
  };
  if constexpr (WHOLE) {
    f32x16 pacc[HALVES];
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int st = 0; st < HALVES; st++) {
      pacc[st] = zero;
      scores(st, pacc[st]);
#pragma unroll
      for (int r = 0; r < 16; r++) { num = fmaf(sacc[st][r], pacc[st][r], num); den += sacc[st][r]; }
    }
    num += __shfl_xor(num, 32, 64);
    den += __shfl_xor(den, 32, 64);
    if (den > 0.f && den < INFINITY) delta = num / den;
#pragma unroll
    for (int st = 0; st < HALVES; st++) grads(st, pacc[st]);
  } else {
#pragma unroll
    for (int st = 0; st < HALVES; st++) {
      f32x16 pacc = zero;
      scores(st, pacc);
      grads(st, pacc);
    }
  }
}

template <int DHP, bool BIAS, bool DROP> constexpr int var_dq_occ() { return (DHP <= 64 && !DROP && !BIAS) ? 3 : DHP <= 96 ? 2 : 1; }
template <int DHP, int NW, bool BIAS, bool DROP>
__global__ __launch_bounds__(NW * 64, (var_dq_occ<DHP, BIAS, DROP>())) void var_dq_k(VarP p) {
  constexpr int TILE = 2 * u_tile<DHP>(), NB = BIAS ? 2 : 3, REQ = 2 * TileDma<DHP, NW>::N;   // see var_fwd_k
  __shared__ __attribute__((aligned(16))) char smem[NB * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = var_block<BIAS>(p, S, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int qrow = hb.xb * (NW * 32) + wid * 32 + (lane & 31);
  const bool qv = qrow < S;
  const bool wave_on = hb.xb * (NW * 32) + wid * 32 < S;
  const bf16* qp = (const bf16*)p.q + b * p.q_sb + h * p.q_sh;
  const bf16* kp = (const bf16*)p.k + b * p.k_sb + h * p.k_sh;
  const bf16* vp = (const bf16*)p.v + b * p.v_sb + h * p.v_sh;
  const bf16* gp = (const bf16*)p.dout + b * p.g_sb + h * p.g_sh;
  const int len = key_count(p, b);
  const uint32_t lds0 = lds_addr(smem);
  const TileDma<DHP, NW> ksrc = tile_dma<DHP, NW>(kp, p.k_ss, len, Dh, lds0, wid, lane);
  const TileDma<DHP, NW> vsrc = tile_dma<DHP, NW>(vp, p.v_ss, len, Dh, lds0 + u_tile<DHP>(), wid, lane);
  auto request = [&](int t, int buf) {   
    tile_request(ksrc, t, buf * TILE);
    tile_request(vsrc, t, buf * TILE);
  };
  const int ntiles = (len + 63) >> 6, nfull = len >> 6;
  bf16x8 qf[DHP / 16], gf[DHP / 16], of[DHP / 16];
  load_stationary<DHP>(qf, qp, p.q_ss, qrow, S, Dh, lane);
  load_stationary<DHP>(gf, gp, p.g_ss, qrow, S, Dh, lane);
  load_stationary<DHP>(of, (const bf16*)p.o + b * p.o_sb + h * p.o_sh, p.o_ss, qrow, S, Dh, lane);
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  const float m = qv ? p.stat[2 * srow] : 0.f, lr = qv ? p.stat[2 * srow + 1] : -INFINITY;
  const int qt = hb.xb * NW + wid;
  const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc(
      BIAS ? (void*)(p.bias_s + ((int64_t)h * p.nqt + (wave_on ? qt : 0)) * p.nkt * 1024) : nullptr, 0, BIAS ? p.nkt * 2048 : 0, 0x00020000);
  bf16x8 bf[4];
  auto load_bias = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; i++) bf[i] = __builtin_bit_cast(bf16x8, buf_load16(brs, (uint32_t)(t * 4096 + i * 1024 + lane * 16)));
  };
  if (BIAS) load_bias(0);
  request(0, 0);
  if (NB == 3) request(1, 1);
  // delta = rowsum(dO * O), each half-wave holds half of the row
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < DHP / 16; ks++)
#pragma unroll
    for (int j = 0; j < 8; j++) delta += (float)of[ks][j] * (float)gf[ks][j];
  delta += __shfl_xor(delta, 32, 64);
  const float c = p.scale * LOG2E, nmc = -m * c;
  const bool big = BIAS && __any(fabsf(m * c) > BIG_EXP);
  if (qv && lane < 32) p.nl[srow] = nmc + lr;   // for the kernels launched after this one
  float dsum = 0.f;
  const uint32_t rbase = var_drop_xrow(p, (uint64_t)srow, lane);
  const f32x16 zero = ZERO16;
  f32x16 dqacc[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) dqacc[dt] = zero;
  u_wait<NB == 3 ? REQ : 0>();   // the stores above are in the count as well: a longer wait, never a shorter one
  __syncthreads();
  int buf = 0;
  const bool whole = ntiles == 1;
  for (int t = 0; t < nfull && !whole; t++) {
    const char* sK = smem + buf * TILE;
    const int ahead = NB == 3 ? (buf == 0 ? 2 : buf - 1) : buf ^ 1;
    f32x16 sacc[2] = {init_tile<BIAS>(bf[0], bf[1], p.inv_scale), init_tile<BIAS>(bf[2], bf[3], p.inv_scale)};
    if (BIAS) load_bias(t + 1);
    request(t + NB - 1, ahead);
    if (wave_on) var_dq_tile<DHP, 2, false, BIAS, DROP>(p, sK, sK + u_tile<DHP>(), qf, gf, sacc, dqacc, m, nmc, big, delta, dsum, c, t * 64, len, rbase, lane);
    u_wait<NB == 3 ? REQ : 0>();
    __syncthreads();
    buf = buf + 1 == NB ? 0 : buf + 1;
  }
  if (whole && wave_on) {
    if (len > 32) {
      f32x16 sacc[2] = {init_tile<BIAS>(bf[0], bf[1], p.inv_scale), init_tile<BIAS>(bf[2], bf[3], p.inv_scale)};
      var_dq_tile<DHP, 2, true, BIAS, DROP, true>(p, smem, smem + u_tile<DHP>(), qf, gf, sacc, dqacc, m, nmc, big, delta, dsum, c, 0, len, rbase, lane);
    } else {
      f32x16 sacc[1] = {init_tile<BIAS>(bf[0], bf[1], p.inv_scale)};
      var_dq_tile<DHP, 1, true, BIAS, DROP, true>(p, smem, smem + u_tile<DHP>(), qf, gf, sacc, dqacc, m, nmc, big, delta, dsum, c, 0, len, rbase, lane);
    }
  } else if (nfull < ntiles && wave_on) {
    const char* sK = smem + buf * TILE;
    const char* sV = sK + u_tile<DHP>();
    if (len - nfull * 64 > 32) {
      f32x16 sacc[2] = {init_tile<BIAS>(bf[0], bf[1], p.inv_scale), init_tile<BIAS>(bf[2], bf[3], p.inv_scale)};
      var_dq_tile<DHP, 2, true, BIAS, DROP>(p, sK, sV, qf, gf, sacc, dqacc, m, nmc, big, delta, dsum, c, nfull * 64, len, rbase, lane);
    } else {
      f32x16 sacc[1] = {init_tile<BIAS>(bf[0], bf[1], p.inv_scale)};
      var_dq_tile<DHP, 1, true, BIAS, DROP>(p, sK, sV, qf, gf, sacc, dqacc, m, nmc, big, delta, dsum, c, nfull * 64, len, rbase, lane);
    }
  }
  u_wait<0>();   // nothing may arrive in LDS after the workgroup has left
  // The rows of dS sum to zero; what they do sum to is the error that O's and P's rounding left in delta, and the kernels that
  // follow get delta without it.  A bias shows it where its buckets hold most of a row's weight (ViT-g/14 at 1024 px with
  // logarithmic buckets: relative error of dtable 2.5e-3 -> 1.7e-3, for 8% of this kernel's time); without one it stays
  // below the rounding of dS.
  if (BIAS) dsum += __shfl_xor(dsum, 32, 64);
  if (!qv) return;
  if (lane < 32) p.delta[srow] = BIAS && lr != -INFINITY ? -fmaf(dsum, fast_exp2(lr), delta) : -delta;
  store_rows<DHP>((bf16*)p.dq + b * p.dq_sb + h * p.dq_sh + (int64_t)qrow * p.dq_ss, dqacc, p.scale * fast_exp2(lr), Dh, lane);
}

// ---- dK, dV -----------------------------------------------------------------------------------------------------------------
// Constants of a tile's 64 query rows: sL = nl = -m c + lr [64], -delta [64], with a bias also (m, lr) [64] (zeros beyond Lq:
// the rows of Q and dO are zeros there, and so is everything they add).  P of a 32 x 32 tile (query r on the accumulator row,
// key on the lane) from its scores; `big`: the tile's rows hold an |m c| beyond BIG_EXP.
template <bool BIAS>
__device__ __forceinline__ void prob_rows(f32x16& sacc, const float* sL, int st, int rowoff, float c, bool big) {
  if (BIAS && big) {
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const float* ml = sL + 128 + 2 * (st * 32 + acc_row(r) + rowoff);
      sacc[r] = fast_exp2((sacc[r] - ml[0]) * c + ml[1]);
    }
  } else {
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const f32x4 n4 = *(const f32x4*)(sL + st * 32 + 8 * g + rowoff);
#pragma unroll
      for (int j = 0; j < 4; j++) sacc[4 * g + j] = fast_exp2(fmaf(sacc[4 * g + j], c, n4[j]));
    }
  }
}
template <bool BIAS> constexpr int row_bytes() { return BIAS ? 1024 : 512; }
// One wave's request for the constants, 256 bytes: nl, delta and the two halves of (m, lr); without a bias waves 2 and 3
// repeat the first two, so that every wave has the same number of requests.
struct RowDma { __amdgpu_buffer_rsrc_t rs; uint32_t dst, row_bytes, off; };
template <bool BIAS> __device__ __forceinline__ RowDma row_dma(const VarP& p, int64_t sbase, uint32_t dst, int wid) {
  RowDma r;
  const bool st = BIAS && wid >= 2;
  const float* src = st ? p.stat + 2 * sbase : (wid & 1 ? p.delta : p.nl) + sbase;
  r.row_bytes = st ? 8u : 4u;
  r.off = st && wid == 3 ? 256u : 0u;
  r.rs = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, p.Lq * (int)r.row_bytes, 0x00020000);
  r.dst = dst + (uint32_t)(BIAS ? wid : wid & 1) * 256u;
  return r;
}
__device__ __forceinline__ void row_request(const RowDma& r, int row0, uint32_t buf_off, int lane) {
  u_dma4(r.rs, (uint32_t)row0 * r.row_bytes + (uint32_t)lane * 4u + r.off, r.dst + buf_off);
}
// Which of the 64 rows hold an |m c| beyond BIG_EXP; from LDS: a load from memory here would wait for every request in flight
// (the counter is one for all), a tile's time each step.
template <bool BIAS> __device__ __forceinline__ uint64_t rows_big(const float* sL, float c, int lane) {
  return BIAS ? __ballot(fabsf(sL[128 + 2 * lane] * c) > BIG_EXP) : 0ull;
}
// dP starts from -delta: P (dP - delta) is then one product (with dropout delta must not be scaled, and is subtracted later)
template <bool DROP> __device__ __forceinline__ f32x16 init_dp(const float* sL, int st, int rowoff) {
  f32x16 a = ZERO16;
  if (!DROP) {
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const f32x4 d4 = *(const f32x4*)(sL + 64 + st * 32 + 8 * g + rowoff);
#pragma unroll
      for (int j = 0; j < 4; j++) a[4 * g + j] = d4[j];
    }
  }
  return a;
}
// dS (in pacc) and the P that multiplies dO (in sacc) of a 32 x 32 tile
template <bool DROP>
__device__ __forceinline__ void ds_rows(const VarP& p, f32x16& sacc, f32x16& pacc, const float* sL, int st, int rowoff,
                                        uint32_t xkey, uint32_t xstep, bool kodd, int khalf) {
#pragma unroll
  for (int g = 0; g < 4; g++) {
    f32x4 d4 = {0.f, 0.f, 0.f, 0.f};
    if (DROP) d4 = *(const f32x4*)(sL + 64 + st * 32 + 8 * g + rowoff);
    uint32_t drops[4] = {0u, 0u, 0u, 0u};
    if (DROP) {   // neighbouring lanes share a pair's hash: each computes two rows' hashes and they swap (see attn.hip)
#pragma unroll
      for (int jj = 0; jj < 2; jj++) {
        const uint32_t mine = rng_fmix(xkey + (uint32_t)(st * 32 + 8 * g + 2 * jj) * xstep);
        const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)mine, 0xB1, 0xF, 0xF, true);   // quad_perm [1,0,3,2]
        const uint32_t h0 = kodd ? other : mine, h1 = kodd ? mine : other;
        drops[2 * jj] = (h0 << khalf) & 0xffff0000u;
        drops[2 * jj + 1] = (h1 << khalf) & 0xffff0000u;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int r = 4 * g + j;
      const float pr = sacc[r];
      float dp = pacc[r];
      if (DROP) {
        const bool keep = drops[j] >= p.thr;
        sacc[r] = keep ? pr * p.keep_scale : 0.f;
        dp = keep ? dp * p.keep_scale : 0.f;
      }
      pacc[r] = pr * (DROP ? dp + d4[j] : dp);
    }
  }
}
struct DropKey { uint32_t xstep; bool kodd; int khalf; uint32_t xk; };
__device__ __forceinline__ DropKey drop_key(const VarP& p, int krow) {
  DropKey d;
  d.xstep = (uint32_t)(var_drop_ld(p) >> 1) * RNG_C1;
  d.kodd = krow & 1;
  d.khalf = d.kodd ? 0 : 16;
  d.xk = (uint32_t)(krow >> 1) * RNG_C1 + rng_seedmix(p.seed);
  return d;
}
__device__ __forceinline__ uint32_t drop_xkey(const VarP& p, const DropKey& d, int64_t row0, int rowoff) {
  return (uint32_t)((uint64_t)(row0 + rowoff + (d.kodd ? 1 : 0)) * (var_drop_ld(p) >> 1)) * RNG_C1 + d.xk;
}

template <int DHP, int HALVES, bool BIAS, bool DROP>
__device__ __forceinline__ void var_dkdv_tile(const VarP& p, const char* sQ, const char* sG, const float* sL,
                                              const bf16x8 (&kf)[DHP / 16], const bf16x8 (&vf)[DHP / 16], bf16x8 (&bf)[4],
                                              __amdgpu_buffer_rsrc_t brs, uint32_t bias_next, f32x16 (&dkacc)[DHP / 32],
                                              f32x16 (&dvacc)[DHP / 32], float c, int64_t bh, int q0, const DropKey& dk, int lane) {
  const int64_t row0 = bh * p.Lq + q0;
  const int rowoff = 4 * (lane >> 5);
  const uint32_t xkey = DROP ? drop_xkey(p, dk, row0, rowoff) : 0u;
  const uint64_t big = rows_big<BIAS>(sL, c, lane);
#pragma unroll
  for (int st = 0; st < HALVES; st++) {
    // a half's bias becomes its initial scores and the registers take the next tile's
    f32x16 sacc = init_tile<BIAS>(bf[2 * st], bf[2 * st + 1], p.inv_scale), pacc = init_dp<DROP>(sL, st, rowoff);
    if (BIAS) {
      bf[2 * st] = __builtin_bit_cast(bf16x8, buf_load16(brs, bias_next + (uint32_t)(st * 2048 + lane * 16)));
      bf[2 * st + 1] = __builtin_bit_cast(bf16x8, buf_load16(brs, bias_next + (uint32_t)(st * 2048 + 1024 + lane * 16)));
    }
#pragma unroll
    for (int ks = 0; ks < DHP / 16; ks++) {
      sacc = MFMA(u_rows<DHP>(sQ, st * 32, ks, lane), kf[ks], sacc, 0, 0, 0);
      pacc = MFMA(u_rows<DHP>(sG, st * 32, ks, lane), vf[ks], pacc, 0, 0, 0);
    }
    prob_rows<BIAS>(sacc, sL, st, rowoff, c, (uint32_t)(big >> (32 * st)) != 0u);
    ds_rows<DROP>(p, sacc, pacc, sL, st, rowoff, xkey, dk.xstep, dk.kodd, dk.khalf);
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      const bf16x8 pf = acc_to_frag(sacc, s2);
      const bf16x8 df = acc_to_frag(pacc, s2);
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++) {
        dvacc[dt] = MFMA(u_cols<DHP>(sG, st * 32, s2, dt * 32, lane), pf, dvacc[dt], 0, 0, 0);
        dkacc[dt] = MFMA(u_cols<DHP>(sQ, st * 32, s2, dt * 32, lane), df, dkacc[dt], 0, 0, 0);
      }
    }
    // two halves in flight at once do not fit beside the accumulators of the larger heads
    if (DHP > 64) __builtin_amdgcn_sched_barrier(0);
  }
}

template <int DHP, bool BIAS, bool DROP> constexpr int var_dkdv_occ() { return (DHP <= 64 || (DHP <= 96 && !DROP)) ? 2 : 1; }
template <int DHP, int NW, bool BIAS, bool DROP>
__global__ __launch_bounds__(NW * 64, (var_dkdv_occ<DHP, BIAS, DROP>())) void var_dkdv_k(VarP p) {
  static_assert(NW == 4, "row_dma");
  constexpr int TILE = 2 * u_tile<DHP>() + row_bytes<BIAS>(), NB = BIAS ? 2 : 3, REQ = 2 * TileDma<DHP, NW>::N + 1;   // Q, dO, row constants; see var_fwd_k
  __shared__ __attribute__((aligned(16))) char smem[NB * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = var_block<BIAS>(p, p.Lk, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h, bh = b * p.H + h;
  const int key0 = hb.xb * (NW * 32), krow = key0 + wid * 32 + (lane & 31);
  const int len = key_count(p, b);
  const bool wave_on = key0 + wid * 32 < len;
  const f32x16 zero = ZERO16;
  f32x16 dkacc[DHP / 32], dvacc[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) { dkacc[dt] = zero; dvacc[dt] = zero; }
  if (key0 < len) {   // otherwise all of the block's keys are padding
    const uint32_t lds0 = lds_addr(smem);
    const TileDma<DHP, NW> qsrc = tile_dma<DHP, NW>((const bf16*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, S, Dh, lds0, wid, lane);
    const TileDma<DHP, NW> gsrc = tile_dma<DHP, NW>((const bf16*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, S, Dh, lds0 + u_tile<DHP>(), wid, lane);
    const RowDma rsrc = row_dma<BIAS>(p, bh * p.Lq, lds0 + 2 * u_tile<DHP>(), wid);
    auto request = [&](int t, int buf) {   
      tile_request(qsrc, t, buf * TILE);
      tile_request(gsrc, t, buf * TILE);
      row_request(rsrc, t * 64, buf * TILE, lane);
    };
    const int ntiles = (S + 63) >> 6, nfull = S >> 6;
    bf16x8 kf[DHP / 16], vf[DHP / 16];
    load_stationary<DHP>(kf, (const bf16*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, krow, len, Dh, lane);
    load_stationary<DHP>(vf, (const bf16*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, krow, len, Dh, lane);
    const int kt = hb.xb * NW + wid;
    const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc(
        BIAS ? (void*)(p.bias_t + ((int64_t)h * p.nkt_t + (wave_on ? kt : 0)) * p.nqt_t * 1024) : nullptr, 0, BIAS ? p.nqt_t * 2048 : 0, 0x00020000);
    bf16x8 bf[4];
    if (BIAS) {
#pragma unroll
      for (int i = 0; i < 4; i++) bf[i] = __builtin_bit_cast(bf16x8, buf_load16(brs, (uint32_t)(i * 1024 + lane * 16)));
    }
    const float c = p.scale * LOG2E;
    const DropKey dkey = drop_key(p, krow);
    request(0, 0);
    if (NB == 3) request(1, 1);
    u_wait<NB == 3 ? REQ : 0>();
    __syncthreads();
    int buf = 0;
    for (int t = 0; t < nfull; t++) {
      const char* sQ = smem + buf * TILE;
      const int ahead = NB == 3 ? (buf == 0 ? 2 : buf - 1) : buf ^ 1;
      request(t + NB - 1, ahead);
      if (wave_on)
        var_dkdv_tile<DHP, 2, BIAS, DROP>(p, sQ, sQ + u_tile<DHP>(), (const float*)(sQ + 2 * u_tile<DHP>()), kf, vf, bf, brs,
                                          (uint32_t)(t + 1) * 4096u, dkacc, dvacc, c, bh, t * 64, dkey, lane);
      u_wait<NB == 3 ? REQ : 0>();
      __syncthreads();
      buf = buf + 1 == NB ? 0 : buf + 1;
    }
    if (nfull < ntiles && wave_on) {
      const char* sQ = smem + buf * TILE;
      const char* sG = sQ + u_tile<DHP>();
      const float* sL = (const float*)(sQ + 2 * u_tile<DHP>());
      const uint32_t none = OOB_OFF;
      if (S - nfull * 64 > 32) var_dkdv_tile<DHP, 2, BIAS, DROP>(p, sQ, sG, sL, kf, vf, bf, brs, none, dkacc, dvacc, c, bh, nfull * 64, dkey, lane);
      else var_dkdv_tile<DHP, 1, BIAS, DROP>(p, sQ, sG, sL, kf, vf, bf, brs, none, dkacc, dvacc, c, bh, nfull * 64, dkey, lane);
    }
    u_wait<0>();   // nothing may arrive in LDS after the workgroup has left
  }
  if (krow >= p.Lk) return;
  bf16* dvp = (bf16*)p.dv + b * p.dv_sb + h * p.dv_sh + (int64_t)krow * p.dv_ss;
  bf16* dkp = (bf16*)p.dk + b * p.dk_sb + h * p.dk_sh + (int64_t)krow * p.dk_ss;
  if (krow >= len) {   // padding: its columns hold whatever the zero rows gave
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) { dkacc[dt] = zero; dvacc[dt] = zero; }
  }
  store_rows<DHP>(dvp, dvacc, 1.f, Dh, lane);
  store_rows<DHP>(dkp, dkacc, p.scale, Dh, lane);
}

// ---- bias gradient: dS summed over the samples ---------------------------------------------------------------------------------
// A workgroup owns 128 keys x 64 queries of a head, 32 x 64 per wave with the key on the lane, and walks the samples of its
// share (p.splits shares); dS of every sample is added to two accumulator tiles per wave, in 32 bits, and leaves as 32-bit
// values.  It forms S' and dP once more, 4 of the 14 products of a training pass, which costs less than writing dS (2 bytes
// per sample, head and pair) and reading it back.  A sample brings 128 rows of K and V and 64 of Q and dO by DMA: the former
// go to registers, which frees their place at once for the next sample's, the latter have NB places: two, or one where two
// would not leave room for a second workgroup on the CU, which matters more (it works while this one starts, waits or
// stores).  ViT-B/14: 131 us with the keys in registers a sample ahead instead of LDS, 61 us so; ViT-g/14 at 1024 px, 4 samples:
// 2.29 ms with one workgroup of 128 queries and two places, 2.08-2.14 ms with two of 64.
template <int DHP> constexpr int dbias_nb() { return DHP == 96 ? 1 : 2; }
template <int DHP, bool DROP>
__global__ __launch_bounds__(256, (DHP <= 96 ? 2 : 1)) void var_dbias_k(VarP p) {
  constexpr int NB = dbias_nb<DHP>();
  constexpr int T = u_tile<DHP>(), KV = 4 * T, QG = 2 * T + row_bytes<true>();   // K, V; Q and dO and the row constants
  __shared__ __attribute__((aligned(16))) char smem[KV + NB * QG];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh;
  const int nkb = (p.Lk + 127) / 128, nqb = (p.Lq + 63) / 64;
  // Neighbours: panels of up to 8 key blocks, all query blocks of a panel, then the next panel of the head (and share): the
  // workgroups that run on an XCD at a time then read few rows between them, which stay in its L2.
  const int64_t it = xcd_item(blockIdx.x, (int64_t)nkb * nqb * p.splits * p.H);
  if (it < 0) return;
  const int64_t hp = it / ((int64_t)nkb * nqb);
  const int part = (int)(hp % p.splits), h = (int)(hp / p.splits), in = (int)(it - hp * nkb * nqb);
  const int panel = in / (8 * nqb), width = min(8, nkb - panel * 8), rest = in - panel * 8 * nqb;
  const int kb = panel * 8 + rest % width, qb = rest / width;
  const int key0 = kb * 128, q0 = qb * 64, krow = key0 + wid * 32 + (lane & 31);
  const int share = (p.B + p.splits - 1) / p.splits;
  const int b_end = min(p.B, share * (part + 1));
  const float c = p.scale * LOG2E;
  const int rowoff = 4 * (lane >> 5);
  const f32x16 zero = ZERO16;
  f32x16 acc[2] = {zero, zero};
  auto next_live = [&](int b) { while (b < b_end && key_count(p, b) <= key0) b++; return b; };
  const int kt = key0 / 32 + wid;   // may lie beyond the last key tile, as the queries may: the descriptor then covers nothing
  const bool tile_on = kt < p.nkt_t && q0 < p.Lq;
  const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p.bias_t + (((int64_t)h * p.nkt_t + (tile_on ? kt : 0)) * p.nqt_t + (tile_on ? q0 / 32 : 0)) * 1024), 0, tile_on ? 4096 : 0, 0x00020000);
  bf16x8 bf[4];   // the same for every sample
#pragma unroll
  for (int i = 0; i < 4; i++) bf[i] = __builtin_bit_cast(bf16x8, buf_load16(brs, (uint32_t)(i * 1024 + lane * 16)));
  const DropKey dkey = drop_key(p, krow);
  const uint32_t lds0 = lds_addr(smem);
  // the same offsets in every sample, another descriptor
  const uint32_t qdst = lds0 + KV;
  const bf16* kh = (const bf16*)p.k + h * p.k_sh;
  const bf16* vh = (const bf16*)p.v + h * p.v_sh;
  const bf16* qh = (const bf16*)p.q + h * p.q_sh;
  const bf16* gh = (const bf16*)p.dout + h * p.g_sh;
  TileDma<DHP, 4> ksrc = tile_dma<DHP, 4>(kh, p.k_ss, p.Lk, Dh, lds0, wid, lane);
  TileDma<DHP, 4> vsrc = tile_dma<DHP, 4>(vh, p.v_ss, p.Lk, Dh, lds0 + 2 * T, wid, lane);
  TileDma<DHP, 4> qsrc = tile_dma<DHP, 4>(qh, p.q_ss, p.Lq, Dh, qdst, wid, lane);
  TileDma<DHP, 4> gsrc = tile_dma<DHP, 4>(gh, p.g_ss, p.Lq, Dh, qdst + T, wid, lane);
  RowDma rsrc = row_dma<true>(p, h * (int64_t)p.Lq, qdst + 2 * T, wid);
  const float* rh = (wid >= 2 ? p.stat + 2 * (h * (int64_t)p.Lq) : (wid & 1 ? p.delta : p.nl) + h * (int64_t)p.Lq);
  const uint32_t rstep = (uint32_t)(p.H * p.Lq) * (wid >= 2 ? 2u : 1u);   // floats from sample to sample
  auto request_keys = [&](int b) {
    const int len = key_count(p, b);
    ksrc.rs = rows_rsrc(kh + (uint32_t)b * p.k_sb, p.k_ss, len, Dh);
    vsrc.rs = rows_rsrc(vh + (uint32_t)b * p.v_sb, p.v_ss, len, Dh);
    ksrc.last = vsrc.last = (len - 1) >> 6;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      tile_request(ksrc, kb * 2 + i, i * T);
      tile_request(vsrc, kb * 2 + i, i * T);
    }
  };
  auto request_rows = [&](int b, int buf) {
    qsrc.rs = rows_rsrc(qh + (uint32_t)b * p.q_sb, p.q_ss, p.Lq, Dh);
    gsrc.rs = rows_rsrc(gh + (uint32_t)b * p.g_sb, p.g_ss, p.Lq, Dh);
    tile_request(qsrc, qb, buf * QG);
    tile_request(gsrc, qb, buf * QG);
    rsrc.rs = __builtin_amdgcn_make_buffer_rsrc((void*)(rh + (uint64_t)(uint32_t)b * rstep), 0, p.Lq * (int)rsrc.row_bytes, 0x00020000);
    row_request(rsrc, q0, buf * QG, lane);
  };
  int b = next_live(share * part), buf = 0;
  if (b < b_end) {
    request_keys(b);
    request_rows(b, 0);
  }
  while (b < b_end) {
    const int len = key_count(p, b), bn = next_live(b + 1);
    const bool wave_on = q0 < p.Lq && key0 + wid * 32 < len, whole = key0 + wid * 32 + 32 <= len, live = krow < len;
    const int64_t bh = (int64_t)b * p.H + h;
    u_wait<0>();
    __syncthreads();
    bf16x8 kf[DHP / 16], vf[DHP / 16];
    {
      const char* sK = smem + (wid >> 1) * T;
#pragma unroll
      for (int ks = 0; ks < DHP / 16; ks++) {
        kf[ks] = u_rows<DHP>(sK, (wid & 1) * 32, ks, lane);
        vf[ks] = u_rows<DHP>(sK + 2 * T, (wid & 1) * 32, ks, lane);
      }
    }
    if (NB == 2 && bn < b_end) request_rows(bn, buf ^ 1);
    __syncthreads();   // every wave has its keys and values
    if (bn < b_end) request_keys(bn);
    if (wave_on) {
      const char* sQ = smem + KV + buf * QG;
      const char* sG = sQ + T;
      const float* sL = (const float*)(sQ + 2 * T);
      const uint32_t xkey = DROP ? drop_xkey(p, dkey, bh * p.Lq + q0, rowoff) : 0u;
      const uint64_t big = rows_big<true>(sL, c, lane);
#pragma unroll
      for (int st = 0; st < 2; st++) {
        f32x16 sacc = init_tile<true>(bf[2 * st], bf[2 * st + 1], p.inv_scale), pacc = init_dp<DROP>(sL, st, rowoff);
#pragma unroll
        for (int ks = 0; ks < DHP / 16; ks++) {
          sacc = MFMA(u_rows<DHP>(sQ, st * 32, ks, lane), kf[ks], sacc, 0, 0, 0);
          pacc = MFMA(u_rows<DHP>(sG, st * 32, ks, lane), vf[ks], pacc, 0, 0, 0);
        }
        prob_rows<true>(sacc, sL, st, rowoff, c, (uint32_t)(big >> (32 * st)) != 0u);
        if (DROP) ds_rows<true>(p, sacc, pacc, sL, st, rowoff, xkey, dkey.xstep, dkey.kodd, dkey.khalf);
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float t = DROP ? acc[st][r] + pacc[r] : fmaf(sacc[r], pacc[r], acc[st][r]);
          acc[st][r] = whole || live ? t : acc[st][r];
        }
      }
    }
    if (NB == 2) buf ^= 1;
    else {
      __syncthreads();
      if (bn < b_end) request_rows(bn, 0);
    }
    b = bn;
  }
  if (krow >= p.Lk) return;
  float* out = p.dbias + ((int64_t)part * p.H + h) * p.Lq * p.Lk + krow;
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int row = q0 + i * 32 + acc_row(r) + rowoff;
      if (row < p.Lq) out[(int64_t)row * p.Lk] = acc[i][r];
    }
}

// ---- up to 32 queries -------------------------------------------------------------------------------------------------------------
// Bound by K, V in and dK, dV out (256 samples x 12 heads of 64, one query over up to 272 states: 90 us for 320 MB, 3.5 TB/s:
// nothing is on its way while a workgroup computes, vector instructions are issued in 43 % of the cycles), so K and V are read
// once: a wave holds 32 keys, forms S' and dP both ways (the query rows' fragments serve as either operand), and writes dK, dV of
// its keys; dQ^T += K^T dS^T of the workgroup's 128 keys goes to p.part and is summed over the key blocks, in their order, by
// var_few_sum_k.
template <int DHP, int STRIDE>
__device__ __forceinline__ void frags_to_lds(const bf16x8 (&f)[DHP / 16], char* s, int lane) {
  const int row = lane & 31, hi = lane >> 5;
#pragma unroll
  for (int ks = 0; ks < DHP / 16; ks++) *(bf16x8*)(s + row * STRIDE + (((ks * 2) | hi) ^ swz_of<1>(row)) * 16) = f[ks];
}
template <int DHP, bool BIAS>
__global__ __launch_bounds__(256, (DHP <= 96 ? 2 : 1)) void var_few_bwd_k(VarP p) {
  constexpr int QS = Strides<DHP>::COLS;
  constexpr int RED = 4 * 32 * (DHP + 4) * 4;   // dQ of the four waves
  constexpr int LDS = 6 * 32 * QS > RED ? 6 * 32 * QS : RED;
  __shared__ __attribute__((aligned(16))) char smem[LDS];   // K of each wave, Q, dO; then the dQ sums
  __shared__ __attribute__((aligned(16))) float sC[4][32];  // -m c + lr, delta, m, lr
  __shared__ float sR[8][32];   // sums of P dP and of P of each wave's keys
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, rowoff = 4 * (lane >> 5);
  const HeadBlock hb = var_block<BIAS>(p, p.Lk, 128);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int len = key_count(p, b), key0 = hb.xb * 128, krow = key0 + wid * 32 + (lane & 31);
  bf16* dvp = (bf16*)p.dv + b * p.dv_sb + h * p.dv_sh + (int64_t)krow * p.dv_ss;
  bf16* dkp = (bf16*)p.dk + b * p.dk_sb + h * p.dk_sh + (int64_t)krow * p.dk_ss;
  const f32x16 zero = ZERO16;
  f32x16 dk[DHP / 32], dv[DHP / 32], dq[DHP / 32];
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; dq[dt] = zero; }
  const int qrow = lane & 31;
  const bool qv = qrow < p.Lq;
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  if (key0 < len) {   // otherwise padding only: zeros to dK and dV, nothing to dQ (var_few_sum_k does not read it)
    bf16x8 kf[DHP / 16], vf[DHP / 16], qf[DHP / 16], gf[DHP / 16];
    load_stationary<DHP>(kf, (const bf16*)p.k + b * p.k_sb + h * p.k_sh, p.k_ss, krow, len, Dh, lane);
    load_stationary<DHP>(vf, (const bf16*)p.v + b * p.v_sb + h * p.v_sh, p.v_ss, krow, len, Dh, lane);
    load_stationary<DHP>(qf, (const bf16*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qrow, p.Lq, Dh, lane);
    load_stationary<DHP>(gf, (const bf16*)p.dout + b * p.g_sb + h * p.g_sh, p.g_ss, qrow, p.Lq, Dh, lane);
    float delta = 0.f;
    {
      bf16x8 of[DHP / 16];
      load_stationary<DHP>(of, (const bf16*)p.o + b * p.o_sb + h * p.o_sh, p.o_ss, qrow, p.Lq, Dh, lane);
#pragma unroll
      for (int ks = 0; ks < DHP / 16; ks++)
#pragma unroll
        for (int j = 0; j < 8; j++) delta += (float)of[ks][j] * (float)gf[ks][j];
      delta += __shfl_xor(delta, 32, 64);
    }
    const float m = qv ? p.stat[2 * srow] : 0.f, lr = qv ? p.stat[2 * srow + 1] : -INFINITY;
    const float c = p.scale * LOG2E, nmc = -m * c;
    const bool big = BIAS && __any(fabsf(m * c) > BIG_EXP);
    char* sK = smem + wid * 32 * QS;
    char* sQ = smem + 4 * 32 * QS;
    char* sG = smem + 5 * 32 * QS;
    frags_to_lds<DHP, QS>(kf, sK, lane);
    if (wid == 0) {
      frags_to_lds<DHP, QS>(qf, sQ, lane);
      if (lane < 32) { sC[0][lane] = nmc + lr; sC[2][lane] = m; sC[3][lane] = lr; }
    }
    if (wid == 1) frags_to_lds<DHP, QS>(gf, sG, lane);
    bf16x8 bs[2], bt[2];
    if (BIAS) {
      const int kt = key0 / 32 + wid;
      const bool on = kt < p.nkt_t;
      const bf16* ps = p.bias_s + ((int64_t)h * p.nqt * p.nkt + (on ? kt : 0)) * 1024 + lane * 8;
      const bf16* pt = p.bias_t + ((int64_t)h * p.nkt_t + (on ? kt : 0)) * p.nqt_t * 1024 + lane * 8;
      bs[0] = *(const bf16x8*)ps; bs[1] = *(const bf16x8*)(ps + 512);
      bt[0] = *(const bf16x8*)pt; bt[1] = *(const bf16x8*)(pt + 512);
    }
    __syncthreads();
    // keys on the rows, query on the lane: P and dP, then dS for dQ
    f32x16 st = init_tile<BIAS>(bs[0], bs[1], p.inv_scale), dt_ = zero;
#pragma unroll
    for (int ks = 0; ks < DHP / 16; ks++) {
      st = MFMA(kf[ks], qf[ks], st, 0, 0, 0);
      dt_ = MFMA(vf[ks], gf[ks], dt_, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const float pr = BIAS && big ? fast_exp2((st[r] - m) * c) : fast_exp2(fmaf(st[r], c, nmc));
      st[r] = key0 + wid * 32 + acc_row(r) + rowoff < len ? pr : 0.f;
    }
    // Where the workgroup holds all keys of the row, delta = sum P dP / sum P, free of O's rounding: with a handful of keys
    // that rounding is much of what dS is made of (5 queries over 9 keys: error of dq 3.3e-3, 2.6e-3 so).
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) { num += st[r] != 0.f ? st[r] * dt_[r] : 0.f; den += st[r]; }
    num += __shfl_xor(num, 32, 64);
    den += __shfl_xor(den, 32, 64);
    if (lane < 32) { sR[wid][lane] = num; sR[4 + wid][lane] = den; }
    __syncthreads();
    if (BIAS && p.pstat && wid == 0 && lane < 32 && qv) {   // for var_few_sum_k
      float* at = p.pstat + 2 * ((int64_t)hb.xb * p.B * p.H * p.Lq + srow);
      at[0] = (sR[0][qrow] + sR[1][qrow]) + (sR[2][qrow] + sR[3][qrow]);
      at[1] = (sR[4][qrow] + sR[5][qrow]) + (sR[6][qrow] + sR[7][qrow]);
    }
    if (len <= 128) {
      const float dn = (sR[4][qrow] + sR[5][qrow]) + (sR[6][qrow] + sR[7][qrow]);
      if (dn > 0.f && dn < INFINITY) delta = ((sR[0][qrow] + sR[1][qrow]) + (sR[2][qrow] + sR[3][qrow])) / dn;
    }
    if (wid == 0 && lane < 32) {
      sC[1][lane] = delta;
      if (BIAS && hb.xb == 0 && qv) { p.delta[srow] = -delta; p.nl[srow] = nmc + lr; }   // for the bias gradient
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
#pragma unroll
      for (int r = 8 * s2; r < 8 * s2 + 8; r++) {
        dt_[r] = st[r] != 0.f ? st[r] * (dt_[r] - delta) : 0.f;
        st[r] = dt_[r] - (float)(bf16)dt_[r];
      }
      // dS (P and dS below) as two bf16 operands, value and rest: the matrix units have time here, and the gradients keep the
      // bits of 32-bit arithmetic up to their own rounding (88 -> 92 us at the case above)
      const bf16x8 df = acc_to_frag(dt_, s2), dr = acc_to_frag(st, s2);
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++) {
        const bf16x8 kc = frag_cols<QS, 1>(sK, 0, s2, dt * 32, lane);
        dq[dt] = MFMA(kc, df, dq[dt], 0, 0, 0);
        dq[dt] = MFMA(kc, dr, dq[dt], 0, 0, 0);
      }
    }
    __syncthreads();
    // queries on the rows, key on the lane: P and dS for dV and dK
    {
      f32x16 s = init_tile<BIAS>(bt[0], bt[1], p.inv_scale), d = zero;
#pragma unroll
      for (int ks = 0; ks < DHP / 16; ks++) {
        s = MFMA(qf[ks], kf[ks], s, 0, 0, 0);
        d = MFMA(gf[ks], vf[ks], d, 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int ql = 8 * g + rowoff;
        const f32x4 n4 = *(const f32x4*)(sC[0] + ql), d4 = *(const f32x4*)(sC[1] + ql);
        const f32x4 m4 = *(const f32x4*)(sC[2] + ql), l4 = *(const f32x4*)(sC[3] + ql);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int r = 4 * g + j;
          s[r] = BIAS && big ? fast_exp2((s[r] - m4[j]) * c + l4[j]) : fast_exp2(fmaf(s[r], c, n4[j]));
          d[r] = s[r] * (d[r] - d4[j]);
        }
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; s2++) {
        const bf16x8 pf = acc_to_frag(s, s2), df = acc_to_frag(d, s2);
#pragma unroll
        for (int r = 8 * s2; r < 8 * s2 + 8; r++) { s[r] -= (float)(bf16)s[r]; d[r] -= (float)(bf16)d[r]; }
        const bf16x8 pr = acc_to_frag(s, s2), dr = acc_to_frag(d, s2);
#pragma unroll
        for (int dt = 0; dt < DHP / 32; dt++) {
          const bf16x8 gc = frag_cols<QS, 1>(sG, 0, s2, dt * 32, lane), qc = frag_cols<QS, 1>(sQ, 0, s2, dt * 32, lane);
          dv[dt] = MFMA(gc, pf, dv[dt], 0, 0, 0);
          dv[dt] = MFMA(gc, pr, dv[dt], 0, 0, 0);
          dk[dt] = MFMA(qc, df, dk[dt], 0, 0, 0);
          dk[dt] = MFMA(qc, dr, dk[dt], 0, 0, 0);
        }
      }
    }
    // dQ of the four waves, summed in their order; a lane holds d = dt*32 + 8 g + rowoff + 0..3 of its query
    __syncthreads();
    float* red = (float*)smem;
    const float f = p.scale * fast_exp2(lr);
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        *(float4*)(red + (wid * 32 + qrow) * (DHP + 4) + dt * 32 + 8 * g + rowoff) =
            make_float4(dq[dt][4 * g] * f, dq[dt][4 * g + 1] * f, dq[dt][4 * g + 2] * f, dq[dt][4 * g + 3] * f);
    __syncthreads();
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    for (int i = tid; i < p.Lq * Dh; i += 256) {
      const int q = i / Dh, d = i - q * Dh;
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) a += red[(w * 32 + q) * (DHP + 4) + d];
      p.part[((int64_t)hb.xb * rows + (b * p.H + h) * p.Lq + q) * Dh + d] = a;
    }
  }
  if (krow >= p.Lk) return;
  if (krow >= len) {
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++) { dk[dt] = zero; dv[dt] = zero; }
  }
  store_rows<DHP>(dvp, dv, 1.f, Dh, lane);
  store_rows<DHP>(dkp, dk, p.scale, Dh, lane);
}
// dQ = sum of the key blocks' shares; 16 lanes per row.  Where the bias gradient follows, it gets delta = sum P dP / sum P over all
// key blocks: a bucket adds up, coherently, what O's rounding leaves in rowsum(dO O) (32 queries over 300 keys in 2 buckets,
// values of mean 4: error of table entries of about 1: 0.5, 7e-5 so).
__global__ __launch_bounds__(256) void var_few_sum_k(VarP p) {
  const int64_t rows = (int64_t)p.B * p.H * p.Lq;
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int j = threadIdx.x & 15;
  if (row >= rows || j * 8 >= p.Dh) return;
  const int64_t i = row % p.Lq, h = (row / p.Lq) % p.H, b = row / ((int64_t)p.Lq * p.H);
  const int n = (key_count(p, b) + 127) / 128;
  float a[8];
#pragma unroll
  for (int k = 0; k < 8; k++) a[k] = 0.f;
  for (int s = 0; s < n; s++) {
    const float* src = p.part + ((int64_t)s * rows + row) * p.Dh + j * 8;
    const float4 x = *(const float4*)src, y = *(const float4*)(src + 4);
    a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w; a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
  }
  if (p.pstat && n > 1 && j == 0) {   // one block has it already
    float num = 0.f, den = 0.f;
    for (int s = 0; s < n; s++) {
      const float2 t = *(const float2*)(p.pstat + 2 * (s * rows + row));
      num += t.x;
      den += t.y;
    }
    if (den > 0.f && den < INFINITY) p.delta[row] = -num / den;
  }
  bf16x8 r;
#pragma unroll
  for (int k = 0; k < 8; k++) r[k] = (bf16)a[k];
  *(bf16x8*)((bf16*)p.dq + b * p.dq_sb + h * p.dq_sh + i * p.dq_ss + j * 8) = r;
}

// ---- launches ------------------------------------------------------------------------------------------------------------------------
#define VAR_DH(FN, ...) do { if (p.Dh <= 64) FN<64, __VA_ARGS__>(p, st); else if (p.Dh <= 96) FN<96, __VA_ARGS__>(p, st); else FN<128, __VA_ARGS__>(p, st); } while (0)
template <int DHP, bool BIAS> static void dq_dh(const VarP& p, hipStream_t st) {
  const dim3 grid(var_grid<BIAS>(p, p.Lq, 128));
  if (p.thr) hipLaunchKernelGGL((var_dq_k<DHP, 4, BIAS, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((var_dq_k<DHP, 4, BIAS, false>), grid, dim3(256), 0, st, p);
}
template <int DHP, bool BIAS> static void dkdv_dh(const VarP& p, hipStream_t st) {
  const dim3 grid(var_grid<BIAS>(p, p.Lk, 128));
  if (p.thr) hipLaunchKernelGGL((var_dkdv_k<DHP, 4, BIAS, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((var_dkdv_k<DHP, 4, BIAS, false>), grid, dim3(256), 0, st, p);
}
template <int DHP, bool DROP> static void dbias_dh(const VarP& p, hipStream_t st) {
  const dim3 grid(xcd_grid(ceil_div(p.Lk, 128) * ceil_div(p.Lq, 64) * p.splits * p.H));
  hipLaunchKernelGGL((var_dbias_k<DHP, DROP>), grid, dim3(256), 0, st, p);
}
template <int DHP, bool BIAS> static void few_dh(const VarP& p, hipStream_t st) {
  hipLaunchKernelGGL((var_few_bwd_k<DHP, BIAS>), dim3(var_grid<BIAS>(p, p.Lk, 128)), dim3(256), 0, st, p);
  hipLaunchKernelGGL(var_few_sum_k, dim3((unsigned)ceil_div((int64_t)p.B * p.H * p.Lq, 16)), dim3(256), 0, st, p);
}
void var_launch_dq(const VarP& p, bool bias, hipStream_t st) { if (bias) VAR_DH(dq_dh, true); else VAR_DH(dq_dh, false); }
void var_launch_dkdv(const VarP& p, bool bias, hipStream_t st) { if (bias) VAR_DH(dkdv_dh, true); else VAR_DH(dkdv_dh, false); }
void var_launch_dbias(const VarP& p, hipStream_t st) { if (p.thr) VAR_DH(dbias_dh, true); else VAR_DH(dbias_dh, false); }
void var_launch_few_bwd(const VarP& p, bool bias, hipStream_t st) { if (bias) VAR_DH(few_dh, true); else VAR_DH(few_dh, false); }
