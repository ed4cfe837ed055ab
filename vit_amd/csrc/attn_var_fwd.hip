// Forward pass on the matrix units (bf16, v_mfma_f32_32x32x16_bf16) of attention with a relative position bias and / or key
// counts, and the bias laid out for it.
//
//   workgroup = NW waves x 32 queries (Q in registers), 64-key tiles of K and V arrive in LDS by DMA; S'^T = K Q^T has the keys
//   on the accumulator rows and the query on the lane, so the running maximum is a register reduction and the probabilities
//   are the next product's operand as they stand.  The bias enters as the INITIAL accumulator of the score product: it costs
//   an unpacking and a multiplication by 1 / scale per element and nothing else.
//   Bound by the latency of a wave's chain through a tile (products, maximum, exponentials, conversion, products), which two or
//   three waves per SIMD do not cover: matrix units 15-35 % busy, vector instructions issued in 32-42 % of the cycles, waves
//   waiting 37-52 % of their time, no LDS bank conflicts (counters of the three cases that follow).  ViT-B/14, 64 samples x 12
//   heads of 64, 272 x 272 with bias: 50 us; ViT-g/14 at 1024 px, 4 samples x 16 heads of 88, 5329 x 5329 with bias: 1.03 ms,
//   620 TFLOP/s (676 as the heads are padded to 96); 300 queries over up to 4096 states, 16 x 16 heads of 64: 90 us.  One
//   sample, 100 queries over 4097 states, 12 heads of 64: 16 shares of the keys, 20 us with their joining.
#include "attn_var.h"

// ---- bias in accumulator order ----------------------------------------------------------------------------------------
// T[index[i][j]][h] as tiles of 32 x 32 in the order in which the lanes of an accumulator tile hold them: tile =
// [2 register halves][64 lanes][8 registers], 16 bytes per lane and half, so that a wave fetches a tile with two coalesced
// 16-byte loads per lane.  TR = false: keys on the rows, query on the lane (forward, dQ), tiles ordered [H][query tile][key
// tile]; TR = true: queries on the rows, key on the lane (dK/dV, bias gradient), [H][key tile][query tile].  Gathering once
// per pair and head here, instead of once per pair, head and sample inside the attention, takes the gather (an LDS or L2
// access with its own address per element) out of the inner loops.  Bound by its stores (16 heads x 5329 x 5329: 216 us, 4.2 TB/s;
// both layouts 400 us, 4.5 TB/s, where a launch each took 508).  HV heads are read per access.
template <int HV> struct HeadVec;
template <> struct HeadVec<8> { typedef uint4 t; };
template <> struct HeadVec<4> { typedef uint2 t; };
template <> struct HeadVec<2> { typedef uint32_t t; };
template <> struct HeadVec<1> { typedef uint16_t t; };

template <int HV, bool TR>
__device__ __forceinline__ void expand_tile(const VarP& p, int lt, int rt, bf16* __restrict__ out) {   // tile along the lanes, along the rows
  const int half = (threadIdx.x >> 6) & 1, lane = threadIdx.x & 63, hi = lane >> 5;
  const int nlt = TR ? p.nkt_t : p.nqt, nrt = TR ? p.nqt_t : p.nkt;
  const int64_t tiles = (int64_t)nlt * nrt, tile = (int64_t)lt * nrt + rt;
  const int at_lane = lt * 32 + (lane & 31);
  int n[8];
  bool ok[8];
#pragma unroll
  for (int r = 0; r < 8; r++) {
    const int at_row = rt * 32 + acc_row(8 * half + r) + 4 * hi;
    const int i = TR ? at_row : at_lane, j = TR ? at_lane : at_row;
    ok[r] = i < p.Lq && j < p.Lk;
    n[r] = ok[r] ? p.index[(int64_t)i * p.Lk + j] : 0;
  }
  typedef typename HeadVec<HV>::t V;
  for (int h = 0; h < p.H; h += HV) {
    uint16_t e[8][HV];
#pragma unroll
    for (int r = 0; r < 8; r++) {
      const V v = *(const V*)((const bf16*)p.table + (int64_t)n[r] * p.H + h);
      __builtin_memcpy(e[r], &v, sizeof(V));
    }
#pragma unroll
    for (int hv = 0; hv < HV; hv++) {
      bf16x8 o;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        const float x = clamp_bias((float)__builtin_bit_cast(bf16, e[r][hv]), p.bias_lim);
        o[r] = (bf16)(ok[r] ? x : 0.f);
      }
      *(bf16x8*)(out + (((int64_t)(h + hv) * tiles + tile) * 2 + half) * 512 + lane * 8) = o;
    }
  }
}
// bias_s alone (forward): two waves a tile, two tiles a workgroup.  BOTH (backward): a workgroup lays the same 32 x 32 pairs out
// both ways, two waves each; nqt_t >= nqt, nkt >= nkt_t.
template <int HV, bool BOTH> __global__ __launch_bounds__(256) void var_expand_k(VarP p) {
  const int which = threadIdx.x >> 7, nq = BOTH ? p.nqt_t : p.nqt;
  const int64_t tile = BOTH ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 2 + which;
  if (tile >= (int64_t)nq * p.nkt) return;
  const int qt = (int)(tile / p.nkt), kt = (int)(tile - (int64_t)qt * p.nkt);
  if (BOTH && which) {
    if (kt < p.nkt_t) expand_tile<HV, true>(p, kt, qt, (bf16*)p.bias_t);
  } else if (qt < p.nqt) {
    expand_tile<HV, false>(p, qt, kt, (bf16*)p.bias_s);
  }
}
template <int HV> static void expand_h(const VarP& p, bool both, hipStream_t st) {
  if (both) hipLaunchKernelGGL((var_expand_k<HV, true>), dim3((unsigned)((int64_t)p.nqt_t * p.nkt)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((var_expand_k<HV, false>), dim3((unsigned)ceil_div((int64_t)p.nqt * p.nkt, 2)), dim3(256), 0, st, p);
}
void var_launch_expand(const VarP& p, bool both, hipStream_t st) {
  const uintptr_t at = (uintptr_t)p.table;
  if (p.H % 8 == 0 && at % 16 == 0) expand_h<8>(p, both, st);
  else if (p.H % 4 == 0 && at % 8 == 0) expand_h<4>(p, both, st);
  else if (p.H % 2 == 0 && at % 4 == 0) expand_h<2>(p, both, st);
  else expand_h<1>(p, both, st);
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// The bias of HALVES 32-key tiles as initial accumulators, in units of 1 / scale
template <int HALVES, bool BIAS>
__device__ __forceinline__ void var_init(f32x16 (&sacc)[HALVES], const bf16x8 (&bf)[4], float inv_scale) {
#pragma unroll
  for (int st = 0; st < HALVES; st++)
#pragma unroll
    for (int r = 0; r < 16; r++) sacc[st][r] = BIAS ? (float)bf[2 * st + (r >> 3)][r & 7] * inv_scale : 0.f;
}
// One 64-key tile (HALVES = 2) or its first 32 keys (HALVES = 1) against a wave's 32 queries; sacc starts as the bias.
template <int DHP, int HALVES, bool PARTIAL, bool BIAS, bool DROP>
__device__ __forceinline__ void var_fwd_tile(const VarP& p, const char* sK, const char* sV, const bf16x8 (&qf)[DHP / 16],
                                             f32x16 (&sacc)[HALVES], f32x16 (&oacc)[DHP / 32], f32x16& lacc, float& m, float c,
                                             int k0, int len, uint32_t xrow, int lane) {
  const int rowoff = 4 * (lane >> 5);
#pragma unroll
  for (int st = 0; st < HALVES; st++)
#pragma unroll
    for (int ks = 0; ks < DHP / 16; ks++) sacc[st] = MFMA(u_rows<DHP>(sK, st * 32, ks, lane), qf[ks], sacc[st], 0, 0, 0);
  if (PARTIAL) {   // keys at or beyond the count (only in the last half of the last tile)
#pragma unroll
    for (int r = 0; r < 16; r++)
      if (k0 + (HALVES - 1) * 32 + acc_row(r) + rowoff >= len) sacc[HALVES - 1][r] = -INFINITY;
  }
  float mx = sacc[0][0];
#pragma unroll
  for (int st = 0; st < HALVES; st++)
#pragma unroll
    for (int r = 0; r < 16; r++) mx = fmaxf(mx, sacc[st][r]);
  mx = max_xor32(mx);
  // m only has to keep the exponentials in range: it is moved (and O, l rescaled) when some query's tile maximum exceeds it
  // by more than 2^8 in the exponent.  A row without any score yet has m = -inf.
  if (__any(mx * c > m * c + 8.f)) {
    const float mnew = fmaxf(m, mx);
    const float alpha = m == mnew ? 1.f : fast_exp2((m - mnew) * c);
    lacc[0] *= alpha;   // only element 0 of the sum tile is ever read
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
      for (int r = 0; r < 16; r++) oacc[dt][r] *= alpha;
    m = mnew;
  }
  const float ms = BIAS && m == -INFINITY ? 0.f : m;   // nothing but -inf so far: the exponentials are 0
  if (BIAS && __any(fabsf(ms * c) > BIG_EXP)) {
#pragma unroll
    for (int st = 0; st < HALVES; st++)
#pragma unroll
      for (int r = 0; r < 16; r++) sacc[st][r] = fast_exp2((sacc[st][r] - ms) * c);
  } else {
    const float nmc = -ms * c;
#pragma unroll
    for (int st = 0; st < HALVES; st++)
#pragma unroll
      for (int r = 0; r < 16; r++) sacc[st][r] = fast_exp2(fmaf(sacc[st][r], c, nmc));
  }
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; j++) ones[j] = (bf16)1.f;
  // O^T[d][q] += V^T[d][key] P^T[key][q].  The probabilities are rounded to bf16 to be an operand (half a step, 2^-8); the
  // row sum is taken of the rounded ones, on the matrix unit, so that the weights of a row add up to 1.
#pragma unroll
  for (int st = 0; st < HALVES; st++)
#pragma unroll
    for (int s2 = 0; s2 < 2; s2++) {
      bf16x8 pf = acc_to_frag(sacc[st], s2);
      lacc = MFMA(ones, pf, lacc, 0, 0, 0);
      if (DROP) {   // registers 8 s2 + 0..3 and + 4..7 are two runs of four consecutive keys, each from a multiple of 4
#pragma unroll
        for (int g = 0; g < 2; g++) {
          uint32_t dr[4];
          rng_lin_run<4>(xrow + (uint32_t)((k0 + st * 32 + acc_row(8 * s2 + 4 * g)) >> 1) * RNG_C1, dr);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int r = 8 * s2 + 4 * g + j;
            sacc[st][r] = dr[j] < p.thr ? 0.f : sacc[st][r] * p.keep_scale;
          }
        }
        pf = acc_to_frag(sacc[st], s2);
      }
#pragma unroll
      for (int dt = 0; dt < DHP / 32; dt++)
        oacc[dt] = MFMA(u_cols<DHP>(sV, st * 32, s2, dt * 32, lane), pf, oacc[dt], 0, 0, 0);
    }
}

// A wave's 32 queries of head (b, h): the normalised rows and their statistics, or with SPLIT the shares for var_combine_k.
template <int DHP, bool SPLIT>
__device__ __forceinline__ void var_fwd_store(const VarP& p, const f32x16 (&oacc)[DHP / 32], float l, float m, int64_t b, int64_t h,
                                              int qrow, int share, int lane) {
  if (qrow >= p.Lq) return;
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  if (SPLIT) {
    const int64_t rows = (int64_t)p.B * p.H * p.Lq;
    const int64_t prow = share * rows + srow;
    float* dst = p.part + prow * p.Dh;
#pragma unroll
    for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int d = dt * 32 + 8 * g + 4 * (lane >> 5);
        if (d < p.Dh) *(float4*)(dst + d) = make_float4(oacc[dt][4 * g], oacc[dt][4 * g + 1], oacc[dt][4 * g + 2], oacc[dt][4 * g + 3]);
      }
    if (lane < 32) { p.pstat[2 * prow] = m; p.pstat[2 * prow + 1] = l; }
    return;
  }
  store_rows<DHP>((bf16*)p.o + b * p.o_sb + h * p.o_sh + (int64_t)qrow * p.o_ss, oacc, l == 0.f ? 0.f : 1.f / l, p.Dh, lane);
  if (lane < 32) {
    p.stat[2 * srow] = l == 0.f ? 0.f : m;
    p.stat[2 * srow + 1] = l == 0.f ? -INFINITY : -__log2f(l);
  }
}

// waves per SIMD: what the registers of an instance allow without spilling
template <int DHP, int NW, bool BIAS, bool DROP> constexpr int var_fwd_occ() {
  return DHP <= 64 ? (!BIAS ? 3 : 2) : DHP <= 96 ? 2 : 1;
}

// SPLIT: the keys of a (sample, head) are shared by gridDim.y workgroups; each leaves O unnormalised in 32 bits with its m and
// row sum, and var_combine_k joins them.
template <int DHP, int NW, bool BIAS, bool DROP, bool SPLIT>
__global__ __launch_bounds__(NW * 64, (var_fwd_occ<DHP, NW, BIAS, DROP>())) void var_fwd_k(VarP p) {
  // Buffers: without a bias the requests are the loop's only memory operations, a tile is asked for two steps ahead and
  // waited for with a count; with one the compiler's wait for a bias tile takes everything with it, so one step ahead.
  constexpr int TILE = 2 * u_tile<DHP>(), NB = BIAS ? 2 : 3, REQ = 2 * TileDma<DHP, NW>::N;
  __shared__ __attribute__((aligned(16))) char smem[NB * TILE];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), Dh = p.Dh, S = p.Lq;
  const HeadBlock hb = var_block<BIAS>(p, S, NW * 32);
  if (!hb.valid) return;
  const int64_t b = hb.b, h = hb.h;
  const int qrow = hb.xb * (NW * 32) + wid * 32 + (lane & 31);
  const bool wave_on = hb.xb * (NW * 32) + wid * 32 < S;   // else this wave only helps staging
  const bf16* qp = (const bf16*)p.q + b * p.q_sb + h * p.q_sh;
  const bf16* kp = (const bf16*)p.k + b * p.k_sb + h * p.k_sh;
  const bf16* vp = (const bf16*)p.v + b * p.v_sb + h * p.v_sh;
  // this workgroup's keys: [64 tile0, len)
  const KeyShare share = key_share(key_count(p, b), 64, SPLIT ? p.splits : 1, SPLIT ? (int)blockIdx.y : 0);
  const int tile0 = share.t0, len = share.end, ntiles = share.t1, nfull = tile0 < ntiles ? len >> 6 : ntiles;
  const uint32_t lds0 = lds_addr(smem);
  const TileDma<DHP, NW> ksrc = tile_dma<DHP, NW>(kp, p.k_ss, len, Dh, lds0, wid, lane);
  const TileDma<DHP, NW> vsrc = tile_dma<DHP, NW>(vp, p.v_ss, len, Dh, lds0 + u_tile<DHP>(), wid, lane);
  auto request = [&](int t, int buf) {
    tile_request(ksrc, t, buf * TILE);
    tile_request(vsrc, t, buf * TILE);
  };
  bf16x8 qf[DHP / 16];
  load_stationary<DHP>(qf, qp, p.q_ss, qrow, S, Dh, lane);
  // bias tiles of this wave's query tile; key tiles beyond the row read as zeros
  const int qt = hb.xb * NW + wid;
  const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc(
      BIAS ? (void*)(p.bias_s + ((int64_t)h * p.nqt + (wave_on ? qt : 0)) * p.nkt * 1024) : nullptr, 0, BIAS ? p.nkt * 2048 : 0, 0x00020000);
  bf16x8 bf[4];
  auto load_bias = [&](bf16x8 (&d)[4], int t) {   // t-th 64-key tile: two 32 x 32 tiles
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = __builtin_bit_cast(bf16x8, buf_load16(brs, (uint32_t)(t * 4096 + i * 1024 + lane * 16)));
  };
  if (BIAS) load_bias(bf, tile0);
  if (tile0 < ntiles) {   // requests beyond the last tile bring the last once more
    request(tile0, 0);
    if (NB == 3) request(tile0 + 1, 1);
  }
  const f32x16 zero = ZERO16;
  f32x16 oacc[DHP / 32], lacc = zero;
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) oacc[dt] = zero;
  float m = -INFINITY;
  const float c = p.scale * LOG2E;
  const uint32_t rbase = var_drop_xrow(p, (uint64_t)(b * p.H + h) * p.Lq + (uint64_t)qrow, lane);
  u_wait<NB == 3 ? REQ : 0>();
  __syncthreads();
  int buf = 0;
  for (int t = tile0; t < nfull; t++) {
    const char* sK = smem + buf * TILE;
    const int ahead = NB == 3 ? (buf == 0 ? 2 : buf - 1) : buf ^ 1;   // the buffer read in the step before
    f32x16 sacc[2];
    var_init<2, BIAS>(sacc, bf, p.inv_scale);
    if (BIAS) load_bias(bf, t + 1);
    request(t + NB - 1, ahead);
    if (wave_on) var_fwd_tile<DHP, 2, false, BIAS, DROP>(p, sK, sK + u_tile<DHP>(), qf, sacc, oacc, lacc, m, c, t * 64, len, rbase, lane);
    u_wait<NB == 3 ? REQ : 0>();   // the next tile has arrived
    __syncthreads();
    buf = buf + 1 == NB ? 0 : buf + 1;
  }
  if (nfull < ntiles && wave_on) {
    const char* sK = smem + buf * TILE;
    const char* sV = sK + u_tile<DHP>();
    if (len - nfull * 64 > 32) {
      f32x16 sacc[2];
      var_init<2, BIAS>(sacc, bf, p.inv_scale);
      var_fwd_tile<DHP, 2, true, BIAS, DROP>(p, sK, sV, qf, sacc, oacc, lacc, m, c, nfull * 64, len, rbase, lane);
    } else {
      f32x16 sacc[1];
      var_init<1, BIAS>(sacc, bf, p.inv_scale);
      var_fwd_tile<DHP, 1, true, BIAS, DROP>(p, sK, sV, qf, sacc, oacc, lacc, m, c, nfull * 64, len, rbase, lane);
    }
  }
  u_wait<0>();   // nothing may arrive in LDS after the workgroup has left
  var_fwd_store<DHP, SPLIT>(p, oacc, lacc[0], m, b, h, qrow, (int)blockIdx.y, lane);
}

// Up to 32 queries: bound by K and V in, and what counts is how many bytes are on their way.  Every wave works for itself, on
// a share of the keys of one head, with 32-key tiles in LDS of its own that it asks for NB - 1 steps ahead: no barrier.  The
// HW heads of a workgroup are neighbours, and so are the workgroups of a sample's key range on an XCD: heads whose rows are
// no multiple of a cache line share lines, which are then fetched once.  One query over up to 5329 states, 16 samples x 16 heads
// of 88: 66 us for the 300 MB of K and V it needs (4.5 TB/s) and 5 us to join 16 shares, where workgroups of one head with
// common tiles took 104 + 5; 256 samples x 12 heads of 64 over up to 272 states: 25 us (36 before).
template <int DHP> constexpr int few_buffers() { return DHP == 96 ? 3 : 2; }
template <int DHP, int HW, bool BIAS, bool SPLIT>
__global__ __launch_bounds__(256, (DHP <= 64 ? 2 : 1)) void var_few_fwd_k(VarP p) {
  constexpr int T = 32 * DHP * 2, NB = few_buffers<DHP>(), REQ = 2 * TileDma<DHP, 2>::N, KW = 4 / HW;
  __shared__ __attribute__((aligned(16))) char smem[4 * NB * 2 * T];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), Dh = p.Dh;
  const int groups = p.H / HW, parts = p.splits / KW;   // of heads; of keys
  const uint32_t i = blockIdx.x >> 3, g = uniform(i / groups) * 8 + (blockIdx.x & 7);
  const int64_t b = uniform(g / parts), h = (int)(i % groups) * HW + wid % HW;
  if (b >= p.B) return;
  const int share = (int)(g - (uint32_t)b * parts) * KW + wid / HW;
  const KeyShare part = key_share(key_count(p, b), 32, p.splits, share);
  const int t0 = (int)uniform(part.t0), nt = (int)uniform(part.t1), len = (int)uniform(part.end);   // keys [32 t0, len)
  const int qrow = lane & 31;
  const uint32_t lds0 = lds_addr(smem) + wid * (NB * 2 * T);
  const bf16* kp = (const bf16*)p.k + b * p.k_sb + h * p.k_sh;
  const bf16* vp = (const bf16*)p.v + b * p.v_sb + h * p.v_sh;
  const WaveDma<DHP> ksrc = wave_dma<DHP>(kp, p.k_ss, len, Dh, lds0, lane), vsrc = wave_dma<DHP>(vp, p.v_ss, len, Dh, lds0 + T, lane);
  const __amdgpu_buffer_rsrc_t brs = __builtin_amdgcn_make_buffer_rsrc(BIAS ? (void*)(p.bias_s + h * p.nqt * p.nkt * 1024) : nullptr, 0, BIAS ? p.nkt * 2048 : 0, 0x00020000);
  bf16x8 qf[DHP / 16], bf[4];
  load_stationary<DHP>(qf, (const bf16*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qrow, p.Lq, Dh, lane);
  auto load_bias = [&](int t) {
#pragma unroll
    for (int k = 0; k < 2; k++) bf[k] = __builtin_bit_cast(bf16x8, buf_load16(brs, (uint32_t)(t * 2048 + k * 1024 + lane * 16)));
  };
  auto request = [&](int t, int buf) {
    wave_request(ksrc, t, buf * 2 * T);
    wave_request(vsrc, t, buf * 2 * T);
  };
  if (BIAS) load_bias(t0);
  if (t0 < nt) {
#pragma unroll
    for (int k = 0; k < NB - 1; k++) request(t0 + k, k);
  }
  const f32x16 zero = ZERO16;
  f32x16 oacc[DHP / 32], lacc = zero;
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++) oacc[dt] = zero;
  float m = -INFINITY;
  const float c = p.scale * LOG2E;
  int buf = 0;
  for (int t = t0; t < nt; t++) {
    u_wait<(NB - 2) * REQ>();   // this tile has arrived
    const char* sK = smem + (wid * NB + buf) * 2 * T;
    f32x16 sacc[1];
    var_init<1, BIAS>(sacc, bf, p.inv_scale);
    if (BIAS) load_bias(t + 1);
    u_wait_lds();   // the reads of the tile before, whose place the next one takes
    request(t + NB - 1, buf == 0 ? NB - 1 : buf - 1);
    if (t * 32 + 32 <= len) var_fwd_tile<DHP, 1, false, BIAS, false>(p, sK, sK + T, qf, sacc, oacc, lacc, m, c, t * 32, len, 0u, lane);
    else var_fwd_tile<DHP, 1, true, BIAS, false>(p, sK, sK + T, qf, sacc, oacc, lacc, m, c, t * 32, len, 0u, lane);
    buf = buf + 1 == NB ? 0 : buf + 1;
  }
  u_wait<0>();   // nothing may arrive in LDS after the workgroup has left
  var_fwd_store<DHP, SPLIT>(p, oacc, lacc[0], m, b, h, qrow, share, lane);
}

// Joins the shares of a row: M = max m, O = sum 2^((m - M) c) O_s / sum 2^((m - M) c) l_s.  A wave per row: 16 lanes hold 8
// values each, the four groups of 16 take every fourth share.
template <class T> __global__ __launch_bounds__(256) void var_combine_k(VarP p) {
  const int64_t rows = (int64_t)p.B * p.H * p.Lq;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int j = threadIdx.x & 15, grp = (threadIdx.x >> 4) & 3;
  if (row >= rows) return;
  const float c = p.scale * LOG2E;
  float M = -INFINITY;
#pragma unroll 4
  for (int s = grp; s < p.splits; s += 4) M = fmaxf(M, p.pstat[2 * (s * rows + row)]);
  M = fmaxf(M, __shfl_xor(M, 16, 64));
  M = fmaxf(M, __shfl_xor(M, 32, 64));
  float l = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = 0.f;
  const bool on = j * 8 < p.Dh;
#pragma unroll 4
  for (int s = grp; s < p.splits; s += 4) {
    const int64_t at = s * rows + row;
    const float m = p.pstat[2 * at], w = m == M ? (M == -INFINITY ? 0.f : 1.f) : fast_exp2((m - M) * c);
    l = fmaf(w, p.pstat[2 * at + 1], l);
    if (on) {   // a share without keys holds zeros
      const float4 a = *(const float4*)(p.part + at * p.Dh + j * 8), b = *(const float4*)(p.part + at * p.Dh + j * 8 + 4);
      o[0] = fmaf(w, a.x, o[0]); o[1] = fmaf(w, a.y, o[1]); o[2] = fmaf(w, a.z, o[2]); o[3] = fmaf(w, a.w, o[3]);
      o[4] = fmaf(w, b.x, o[4]); o[5] = fmaf(w, b.y, o[5]); o[6] = fmaf(w, b.z, o[6]); o[7] = fmaf(w, b.w, o[7]);
    }
  }
#pragma unroll
  for (int x = 16; x < 64; x *= 2) {
    l += __shfl_xor(l, x, 64);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] += __shfl_xor(o[i], x, 64);
  }
  if (grp) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t i = row % p.Lq, h = (row / p.Lq) % p.H, b = row / ((int64_t)p.Lq * p.H);
  if (on) {
    T* dst = (T*)p.o + b * p.o_sb + h * p.o_sh + i * p.o_ss + j * 8;
    Vec4<T> x, y;
#pragma unroll
    for (int k = 0; k < 4; k++) { x.v[k] = o[k] * inv; y.v[k] = o[4 + k] * inv; }
    x.store(dst);
    y.store(dst + 4);
  }
  if (j == 0) {
    p.stat[2 * row] = l == 0.f ? 0.f : M;
    p.stat[2 * row + 1] = l == 0.f ? -INFINITY : -__log2f(l);
  }
}

void var_launch_combine(const VarP& p, bool f32, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div((int64_t)p.B * p.H * p.Lq, 4));
  if (f32) hipLaunchKernelGGL((var_combine_k<float>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((var_combine_k<bf16>), grid, dim3(256), 0, st, p);
}
// Heads of a workgroup of var_few_fwd_k; its other waves share keys.
int var_few_heads(int64_t H) { return H % 4 == 0 ? 4 : H % 2 == 0 ? 2 : 1; }
template <int DHP, bool BIAS, int HW> static void few_fwd(const VarP& p, hipStream_t st) {
  const dim3 grid((unsigned)(ceil_div((int64_t)p.B * (p.splits / (4 / HW)), 8) * 8 * (p.H / HW)));
  if constexpr (HW == 4) {
    if (p.splits == 1) {
      hipLaunchKernelGGL((var_few_fwd_k<DHP, HW, BIAS, false>), grid, dim3(256), 0, st, p);
      return;
    }
  }
  hipLaunchKernelGGL((var_few_fwd_k<DHP, HW, BIAS, true>), grid, dim3(256), 0, st, p);
}
template <int DHP, bool BIAS> static void few_fwd_dh(const VarP& p, hipStream_t st) {
  const int hw = var_few_heads(p.H);
  if (hw == 4) few_fwd<DHP, BIAS, 4>(p, st);
  else if (hw == 2) few_fwd<DHP, BIAS, 2>(p, st);
  else few_fwd<DHP, BIAS, 1>(p, st);
  if (p.splits > 1) var_launch_combine(p, false, st);
}
template <int DHP, bool BIAS> static void fwd_dh(const VarP& p, int nw, hipStream_t st) {
  const dim3 grid(var_grid<BIAS>(p, p.Lq, nw * 32), (unsigned)p.splits);
  if (p.thr) {
    hipLaunchKernelGGL((var_fwd_k<DHP, 4, BIAS, true, false>), grid, dim3(256), 0, st, p);
  } else if (p.splits > 1) {
    if (nw == 2) hipLaunchKernelGGL((var_fwd_k<DHP, 2, BIAS, false, true>), grid, dim3(128), 0, st, p);
    else hipLaunchKernelGGL((var_fwd_k<DHP, 4, BIAS, false, true>), grid, dim3(256), 0, st, p);
    var_launch_combine(p, false, st);
  } else {
    if (nw == 2) hipLaunchKernelGGL((var_fwd_k<DHP, 2, BIAS, false, false>), grid, dim3(128), 0, st, p);
    else hipLaunchKernelGGL((var_fwd_k<DHP, 4, BIAS, false, false>), grid, dim3(256), 0, st, p);
  }
}
void var_launch_few_fwd(const VarP& p, bool bias, hipStream_t st) {
  if (p.Dh <= 64) { if (bias) few_fwd_dh<64, true>(p, st); else few_fwd_dh<64, false>(p, st); }
  else if (p.Dh <= 96) { if (bias) few_fwd_dh<96, true>(p, st); else few_fwd_dh<96, false>(p, st); }
  else { if (bias) few_fwd_dh<128, true>(p, st); else few_fwd_dh<128, false>(p, st); }
}
void var_launch_fwd(const VarP& p, bool bias, int nw, hipStream_t st) {
  if (p.Dh <= 64) { if (bias) fwd_dh<64, true>(p, nw, st); else fwd_dh<64, false>(p, nw, st); }
  else if (p.Dh <= 96) { if (bias) fwd_dh<96, true>(p, nw, st); else fwd_dh<96, false>(p, nw, st); }
  else { if (bias) fwd_dh<128, true>(p, nw, st); else fwd_dh<128, false>(p, nw, st); }
}
