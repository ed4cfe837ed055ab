// Attention with a learned relative position bias and / or a key count per sample, forward and backward.
//
//   S = scale Q K^T + T[bucket(i, j), h] over the keys j < len(b),  P = softmax(S),  O = P V
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - rowsum(dO O)),  dQ = scale dS K,  dK = scale dS^T Q,
//   dT[n, h] = sum over samples and over the pairs (i, j) of bucket n of dS
//
// This file: the portable kernels (any dtype, head_dim <= 128, any strides, fp32 math; 64 stationary rows per workgroup, 4
// threads per row), the bucket sums and the entry points.  On the matrix units: attn_var_fwd.hip, attn_var_bwd.hip (bf16),
// attn_var_f32.hip (float32).
#include "attn_var.h"

constexpr int VMAXI = 32;  // head_dim <= 128
constexpr int VT = 32;     // streamed rows per LDS tile

template <class T>
__device__ __forceinline__ void vload_tile(float* dst, const T* src, int64_t ss, int64_t row0, int64_t nrows, int Dh, int tid) {
  for (int i = tid; i < VT * Dh; i += 256) {
    const int r = i / Dh, d = i % Dh;
    dst[i] = (row0 + r < nrows) ? to_f<T>(src[(row0 + r) * ss + d]) : 0.f;
  }
}
__device__ __forceinline__ float vquad_sum(float v) {
  v += __shfl_xor(v, 1, 64);
  v += __shfl_xor(v, 2, 64);
  return v;
}
// bias of a pair in units of 1 / scale
template <class T> __device__ __forceinline__ float var_bias(const VarP& p, int64_t i, int64_t j, int64_t h) {
  return p.table ? clamp_bias(to_f<T>(((const T*)p.table)[(int64_t)p.index[i * p.Lk + j] * p.H + h]), p.bias_lim) * p.inv_scale : 0.f;
}

template <class T>
__global__ __launch_bounds__(256) void var_fwd_simple_k(VarP p) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int Dh = p.Dh, tid = threadIdx.x, part = tid & 3;
  const int64_t b = blockIdx.z, h = blockIdx.y, qrow = (int64_t)blockIdx.x * 64 + (tid >> 2);
  float* Ks = sm;
  float* Vs = sm + VT * Dh;
  const T* qp = (const T*)p.q + b * p.q_sb + h * p.q_sh;
  const T* kp = (const T*)p.k + b * p.k_sb + h * p.k_sh;
  const T* vp = (const T*)p.v + b * p.v_sb + h * p.v_sh;
  const bool qv = qrow < p.Lq;
  const int len = key_count(p, b);
  float q[VMAXI], o[VMAXI];
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    q[i] = (qv && d < Dh) ? to_f<T>(qp[qrow * p.q_ss + d]) : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const float c = p.scale * LOG2E;
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  const uint64_t rbase = (uint64_t)srow * var_drop_ld(p);
  for (int64_t k0 = 0; k0 < len; k0 += VT) {
    __syncthreads();
    vload_tile<T>(Ks, kp, p.k_ss, k0, len, Dh, tid);
    vload_tile<T>(Vs, vp, p.v_ss, k0, len, Dh, tid);
    __syncthreads();
    const int nk = (int)(len - k0 < VT ? len - k0 : VT);
    for (int kk = 0; kk < nk; kk++) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) s = fmaf(q[i], Ks[kk * Dh + d], s);
      }
      s = vquad_sum(s);
      if (qv) s += var_bias<T>(p, qrow, k0 + kk, h);
      if (s == -INFINITY) continue;   // nothing of this key (the whole quad skips together)
      const float mn = fmaxf(m, s);
      const float a = exp2f(__fmul_rn(m - mn, c)), pr = exp2f(__fmul_rn(s - mn, c));
      l = l * a + pr;
      m = mn;
      float pd = pr;
      if (p.thr) pd = rng_u32(p.seed, rbase + (uint64_t)(k0 + kk)) >= p.thr ? pr * p.keep_scale : 0.f;
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) o[i] = fmaf(pd, Vs[kk * Dh + d], o[i] * a);
      }
    }
  }
  if (!qv) return;
  T* op = (T*)p.o + b * p.o_sb + h * p.o_sh + qrow * p.o_ss;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    if (d < Dh) op[d] = from_f<T>(o[i] * inv);
  }
  if (part == 0) { p.stat[2 * srow] = l == 0.f ? 0.f : m; p.stat[2 * srow + 1] = l == 0.f ? -INFINITY : -log2f(l); }
}

// delta[b,h,i] = sum_d dO O   (a wave per row)
template <class T>
__global__ __launch_bounds__(256) void var_delta_k(VarP p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.H * p.Lq) return;
  const int64_t s = row % p.Lq, h = (row / p.Lq) % p.H, b = row / ((int64_t)p.Lq * p.H);
  const T* o = (const T*)p.o + b * p.o_sb + h * p.o_sh + s * p.o_ss;
  const T* g = (const T*)p.dout + b * p.g_sb + h * p.g_sh + s * p.g_ss;
  float acc = 0.f;
  for (int d = lane; d < p.Dh; d += 64) acc += to_f<T>(o[d]) * to_f<T>(g[d]);
  acc = wave_sum(acc);
  if (lane == 0) p.delta[row] = acc;
}

template <class T>
__global__ __launch_bounds__(256) void var_dq_simple_k(VarP p) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int Dh = p.Dh, tid = threadIdx.x, part = tid & 3;
  const int64_t b = blockIdx.z, h = blockIdx.y, qrow = (int64_t)blockIdx.x * 64 + (tid >> 2);
  float* Ks = sm;
  float* Vs = sm + VT * Dh;
  const T* qp = (const T*)p.q + b * p.q_sb + h * p.q_sh;
  const T* kp = (const T*)p.k + b * p.k_sb + h * p.k_sh;
  const T* vp = (const T*)p.v + b * p.v_sb + h * p.v_sh;
  const T* gp = (const T*)p.dout + b * p.g_sb + h * p.g_sh;
  const bool qv = qrow < p.Lq;
  const int len = key_count(p, b);
  float q[VMAXI], g[VMAXI], dq[VMAXI];
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    q[i] = (qv && d < Dh) ? to_f<T>(qp[qrow * p.q_ss + d]) : 0.f;
    g[i] = (qv && d < Dh) ? to_f<T>(gp[qrow * p.g_ss + d]) : 0.f;
    dq[i] = 0.f;
  }
  const int64_t srow = (b * p.H + h) * p.Lq + qrow;
  const float m = qv ? p.stat[2 * srow] : 0.f, lr = qv ? p.stat[2 * srow + 1] : 0.f, delta = qv ? p.delta[srow] : 0.f;
  const float c = p.scale * LOG2E;
  float dsum = 0.f;
  const uint64_t rbase = (uint64_t)srow * var_drop_ld(p);
  for (int64_t k0 = 0; k0 < len; k0 += VT) {
    __syncthreads();
    vload_tile<T>(Ks, kp, p.k_ss, k0, len, Dh, tid);
    vload_tile<T>(Vs, vp, p.v_ss, k0, len, Dh, tid);
    __syncthreads();
    const int nk = (int)(len - k0 < VT ? len - k0 : VT);
    for (int kk = 0; kk < nk; kk++) {
      float s = 0.f, dp = 0.f;
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) { s = fmaf(q[i], Ks[kk * Dh + d], s); dp = fmaf(g[i], Vs[kk * Dh + d], dp); }
      }
      s = vquad_sum(s);
      dp = vquad_sum(dp);
      if (qv) s += var_bias<T>(p, qrow, k0 + kk, h);
      const float pr = exp2f(__fmul_rn(s - m, c) + lr);
      if (p.thr) dp = rng_u32(p.seed, rbase + (uint64_t)(k0 + kk)) >= p.thr ? dp * p.keep_scale : 0.f;
      const float ds = pr * (dp - delta);
      dsum += ds;
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) dq[i] = fmaf(ds, Ks[kk * Dh + d], dq[i]);
      }
    }
  }
  if (!qv) return;
  // The rows of dS sum to zero; what they do sum to is what O's rounding left in delta, and a bucket of the bias gradient would
  // add it up: the kernels that follow get delta without it.
  if (p.table && part == 0) p.delta[srow] = delta + dsum;
  T* op = (T*)p.dq + b * p.dq_sb + h * p.dq_sh + qrow * p.dq_ss;
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    if (d < Dh) op[d] = from_f<T>(dq[i] * p.scale);
  }
}

template <class T>
__global__ __launch_bounds__(256) void var_dkdv_simple_k(VarP p) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  const int Dh = p.Dh, tid = threadIdx.x, part = tid & 3;
  const int64_t b = blockIdx.z, h = blockIdx.y, krow = (int64_t)blockIdx.x * 64 + (tid >> 2);
  float* Qs = sm;
  float* Gs = sm + VT * Dh;
  float* Ls = sm + 2 * VT * Dh;   // m[VT], lr[VT], delta[VT]
  const float c = p.scale * LOG2E;
  const T* qp = (const T*)p.q + b * p.q_sb + h * p.q_sh;
  const T* kp = (const T*)p.k + b * p.k_sb + h * p.k_sh;
  const T* vp = (const T*)p.v + b * p.v_sb + h * p.v_sh;
  const T* gp = (const T*)p.dout + b * p.g_sb + h * p.g_sh;
  const int len = key_count(p, b);
  const bool kv = krow < len;
  float k[VMAXI], v[VMAXI], dk[VMAXI], dv[VMAXI];
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    k[i] = (kv && d < Dh) ? to_f<T>(kp[krow * p.k_ss + d]) : 0.f;
    v[i] = (kv && d < Dh) ? to_f<T>(vp[krow * p.v_ss + d]) : 0.f;
    dk[i] = 0.f; dv[i] = 0.f;
  }
  const int64_t sbase = (b * p.H + h) * p.Lq;
  const bool any = (int64_t)blockIdx.x * 64 < len;   // otherwise the whole block of keys is padding
  for (int64_t q0 = 0; any && q0 < p.Lq; q0 += VT) {
    __syncthreads();
    vload_tile<T>(Qs, qp, p.q_ss, q0, p.Lq, Dh, tid);
    vload_tile<T>(Gs, gp, p.g_ss, q0, p.Lq, Dh, tid);
    if (tid < VT) {
      const bool ok = q0 + tid < p.Lq;
      Ls[tid] = ok ? p.stat[2 * (sbase + q0 + tid)] : 0.f;
      Ls[VT + tid] = ok ? p.stat[2 * (sbase + q0 + tid) + 1] : 0.f;
      Ls[2 * VT + tid] = ok ? p.delta[sbase + q0 + tid] : 0.f;
    }
    __syncthreads();
    const int nq = (int)(p.Lq - q0 < VT ? p.Lq - q0 : VT);
    for (int qq = 0; qq < nq; qq++) {
      float s = 0.f, dp = 0.f;
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) { s = fmaf(k[i], Qs[qq * Dh + d], s); dp = fmaf(v[i], Gs[qq * Dh + d], dp); }
      }
      s = vquad_sum(s);
      dp = vquad_sum(dp);
      if (kv) s += var_bias<T>(p, q0 + qq, krow, h);
      const float pr = kv ? exp2f(__fmul_rn(s - Ls[qq], c) + Ls[VT + qq]) : 0.f;
      float pd = pr;
      if (p.thr) {
        const bool keep = rng_u32(p.seed, (uint64_t)(sbase + q0 + qq) * var_drop_ld(p) + (uint64_t)krow) >= p.thr;
        pd = keep ? pr * p.keep_scale : 0.f;
        dp = keep ? dp * p.keep_scale : 0.f;
      }
      const float ds = pr * (dp - Ls[2 * VT + qq]);
#pragma unroll
      for (int i = 0; i < VMAXI; i++) {
        const int d = part + 4 * i;
        if (d < Dh) { dv[i] = fmaf(pd, Gs[qq * Dh + d], dv[i]); dk[i] = fmaf(ds, Qs[qq * Dh + d], dk[i]); }
      }
    }
  }
  if (krow >= p.Lk) return;
  T* okp = (T*)p.dk + b * p.dk_sb + h * p.dk_sh + krow * p.dk_ss;
  T* ovp = (T*)p.dv + b * p.dv_sb + h * p.dv_sh + krow * p.dv_ss;
#pragma unroll
  for (int i = 0; i < VMAXI; i++) {
    const int d = part + 4 * i;
    if (d < Dh) { okp[d] = from_f<T>(kv ? dk[i] * p.scale : 0.f); ovp[d] = from_f<T>(kv ? dv[i] : 0.f); }
  }
}

// dbias[h][i][j] = sum_b dS   (a thread per pair)
template <class T>
__global__ __launch_bounds__(256) void var_dbias_simple_k(VarP p) {
  const int64_t pair = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t h = blockIdx.y;
  if (pair >= (int64_t)p.Lq * p.Lk) return;
  const int64_t i = pair / p.Lk, j = pair - i * p.Lk;
  const float bias = var_bias<T>(p, i, j, h);
  float sum = 0.f;
  for (int64_t b = 0; b < p.B; b++) {
    if (j >= key_count(p, b)) continue;
    const T* q = (const T*)p.q + b * p.q_sb + h * p.q_sh + i * p.q_ss;
    const T* k = (const T*)p.k + b * p.k_sb + h * p.k_sh + j * p.k_ss;
    const T* v = (const T*)p.v + b * p.v_sb + h * p.v_sh + j * p.v_ss;
    const T* g = (const T*)p.dout + b * p.g_sb + h * p.g_sh + i * p.g_ss;
    float s = 0.f, dp = 0.f;
    for (int d = 0; d < p.Dh; d++) { s = fmaf(to_f<T>(q[d]), to_f<T>(k[d]), s); dp = fmaf(to_f<T>(g[d]), to_f<T>(v[d]), dp); }
    const int64_t srow = (b * p.H + h) * p.Lq + i;
    const float pr = exp2f(__fmul_rn(s + bias - p.stat[2 * srow], p.scale * LOG2E) + p.stat[2 * srow + 1]);
    if (p.thr) dp = rng_u32(p.seed, (uint64_t)srow * var_drop_ld(p) + (uint64_t)j) >= p.thr ? dp * p.keep_scale : 0.f;
    sum += pr * (dp - p.delta[srow]);
  }
  p.dbias[h * p.Lq * p.Lk + pair] = sum;
}

// ---- bucket sums of dbias: pieces of a bucket's pairs, then the pieces of a bucket, both in a fixed order -------------------
// Bound by reading dbias, a value per lane and line (16 heads x 5329 x 5329: 460 us, 4.0 TB/s).  A wave sums one piece for up to
// 4 heads: a pair number is read once for them, and 4 pairs x 4 heads are in flight per lane (ViT-B/14: 61 us a head at a
// time, 13 us so, with neighbouring pieces on one XCD).
__global__ __launch_bounds__(256) void var_piece_sum_k(const float* __restrict__ dbias, const int32_t* __restrict__ order,
                                                       const int32_t* __restrict__ piece, float* __restrict__ part,
                                                       int64_t pairs, int H, int npieces, int splits) {
  // Neighbouring pieces on one XCD: the pairs of a bucket lie along a diagonal, a value per cache line, and the rest of each
  // line belongs to the buckets next to it.
  const int nblk = (npieces + 3) / 4;
  const int64_t it = xcd_item(blockIdx.x, (int64_t)nblk * ((H + 3) / 4));
  if (it < 0) return;
  const int lane = threadIdx.x & 63, pc = (int)(it % nblk) * 4 + (threadIdx.x >> 6), h0 = (int)(it / nblk) * 4;
  if (pc >= npieces) return;
  const int b = piece[pc], e = piece[pc + 1], nh = min(4, H - h0);
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = b + lane; i < e; i += 256) {
    int64_t at[4];
#pragma unroll
    for (int u = 0; u < 4; u++) at[u] = i + 64 * u < e ? order[i + 64 * u] : -1;
#pragma unroll 2
    for (int s = 0; s < splits; s++) {
      const float* src = dbias + ((int64_t)s * H + h0) * pairs;
      float x[4][4];
#pragma unroll
      for (int u = 0; u < 4; u++)
#pragma unroll
        for (int k = 0; k < 4; k++) x[u][k] = at[u] >= 0 && k < nh ? src[k * pairs + at[u]] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; k++) a[k] += (x[0][k] + x[1][k]) + (x[2][k] + x[3][k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const float t = wave_sum(a[k]);
    if (lane == 0 && k < nh) part[(int64_t)(h0 + k) * npieces + pc] = t;
  }
}
// a workgroup per bucket and head
template <class T>
__global__ __launch_bounds__(256) void var_bucket_sum_k(const float* __restrict__ part, const int32_t* __restrict__ bucket_piece,
                                                        T* __restrict__ out, int H, int npieces) {
  __shared__ float red[4];
  const int n = (int)blockIdx.x, h = blockIdx.y, b = bucket_piece[n], e = bucket_piece[n + 1];
  if (e - b <= 1) {   // most buckets of a grid: one piece
    if (threadIdx.x == 0) out[(int64_t)n * H + h] = from_f<T>(e > b ? part[(int64_t)h * npieces + b] : 0.f);
    return;
  }
  float a = 0.f;
  for (int i = b + (int)threadIdx.x; i < e; i += 256) a += part[(int64_t)h * npieces + i];
  a = wave_sum(a);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x == 0) out[(int64_t)n * H + h] = from_f<T>((red[0] + red[1]) + (red[2] + red[3]));
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static VarP make_varp(const VitkAttnVar* a) {
  VarP p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->o; p.dout = a->dout; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
  p.stat = a->stat; p.kv_len = a->kv_len; p.table = a->bias_table; p.index = a->bias_index;
  const int64_t* s = a->st;
  p.q_sb = s[0]; p.q_sh = s[1]; p.q_ss = s[2]; p.k_sb = s[3]; p.k_sh = s[4]; p.k_ss = s[5];
  p.v_sb = s[6]; p.v_sh = s[7]; p.v_ss = s[8]; p.o_sb = s[9]; p.o_sh = s[10]; p.o_ss = s[11];
  p.g_sb = s[12]; p.g_sh = s[13]; p.g_ss = s[14]; p.dq_sb = s[15]; p.dq_sh = s[16]; p.dq_ss = s[17];
  p.dk_sb = s[18]; p.dk_sh = s[19]; p.dk_ss = s[20]; p.dv_sb = s[21]; p.dv_sh = s[22]; p.dv_ss = s[23];
  p.B = (int)a->B; p.H = (int)a->H; p.Lq = (int)a->Lq; p.Lk = (int)a->Lk; p.Dh = (int)a->Dh;
  p.nqt = (int)ceil_div(a->Lq, 32); p.nkt = (int)ceil_div(a->Lk, 64) * 2;
  p.nkt_t = (int)ceil_div(a->Lk, 32); p.nqt_t = (int)ceil_div(a->Lq, 64) * 2;
  p.splits = 1; p.buckets = (int)a->num_buckets;
  p.seed = a->seed; p.scale = a->scale; p.inv_scale = 1.f / a->scale;
  p.bias_lim = 1e38f * a->scale < 1e37f ? 1e38f * a->scale : 1e37f;
  p.thr = a->drop_p > 0.f ? drop_threshold(a->drop_p) : 0;
  p.keep_scale = 1.f / (1.f - a->drop_p);
  return p;
}
// The stride of an axis of one element is never used; torch leaves anything there.
static VitkAttnVar var_normal(const VitkAttnVar* a) {
  VitkAttnVar n = *a;
  for (int i = 0; i < 8; i++) {
    const bool key_side = i == 1 || i == 2 || i == 6 || i == 7;   // q, k, v, o, dout, dq, dk, dv
    if (n.B == 1) n.st[3 * i] = 0;
    if (n.H == 1) n.st[3 * i + 1] = 0;
    if ((key_side ? n.Lk : n.Lq) == 1) n.st[3 * i + 2] = (n.Dh + 7) & ~7;   // the next row lies behind the end: see var_mfma_ok
  }
  return n;
}
static int var_validate(const VitkAttnVar* a, bool bwd) {
  VITK_REQUIRE(a, "attn_var: null descriptor");
  VITK_REQUIRE(a->B >= 0 && a->B <= 65535 && a->H > 0 && a->H <= 65535 && a->Lq >= 0 && a->Lk >= 0 && a->Dh > 0 && a->Dh <= 128,
               "attn_var: bad shape B=%lld H=%lld Lq=%lld Lk=%lld Dh=%lld", (long long)a->B, (long long)a->H, (long long)a->Lq,
               (long long)a->Lk, (long long)a->Dh);
  VITK_REQUIRE(a->Lq < (1 << 22) && a->Lk < (1 << 24), "attn_var: at most 2^22 queries and 2^24 keys");
  VITK_REQUIRE((a->B * a->H + 8) * (ceil_div(a->Lq > a->Lk ? a->Lq : a->Lk, 64) + 1) < (1ll << 31), "attn_var: too many rows for one launch");
  VITK_REQUIRE(a->dtype == VITK_F32 || a->dtype == VITK_BF16, "attn_var: bad dtype");
  VITK_REQUIRE(!a->dbias_table || a->dbias_dtype == VITK_F32 || a->dbias_dtype == VITK_BF16, "attn_var: bad dtype of the bias gradient");
  VITK_REQUIRE(a->drop_p >= 0.f && a->drop_p < 1.f, "attn_var: dropout p=%f out of range", a->drop_p);
  VITK_REQUIRE(a->scale > 1e-30f && a->scale < 1e10f, "attn_var: scale=%g outside (1e-30, 1e10)", a->scale);
  if (a->B * a->Lq * a->Lk > 0) VITK_REQUIRE(a->q && a->k && a->v && a->o && a->stat, "attn_var: null pointer");
  VITK_REQUIRE(!a->bias_table == !a->bias_index, "attn_var: a bias needs its table and its index");
  if (a->bias_table) {
    VITK_REQUIRE(a->num_buckets > 0 && a->num_buckets <= 65536, "attn_var: num_buckets=%lld outside [1, 65536]", (long long)a->num_buckets);
    VITK_REQUIRE(a->num_buckets * a->H < (1ll << 29), "attn_var: a bias table of %lld x %lld is not supported", (long long)a->num_buckets, (long long)a->H);
    VITK_REQUIRE(a->Lq * a->Lk < (1ll << 31), "attn_var: a bias over %lld x %lld pairs is not supported", (long long)a->Lq, (long long)a->Lk);
  }
  if (bwd) {
    VITK_REQUIRE(a->B * a->Lq == 0 || (a->dout && a->dq), "attn_var_bwd: null pointer");
    VITK_REQUIRE(a->B * a->Lk == 0 || (a->dk && a->dv), "attn_var_bwd: null pointer");
    if (a->dbias_table)
      VITK_REQUIRE(a->bias_table && a->order && a->piece && a->bucket_piece && a->num_pieces >= 0, "attn_var_bwd: the bias gradient needs the bias and its plan");
  }
  return 0;
}
// The matrix-unit kernels take head sizes that are multiples of 8, 16-byte aligned rows, and rows of one (sample, head)
// within 32-bit byte offsets (the tiles asked for ahead of the last one included).  Rows have to follow each other: the
// kernels find the rows beyond the last by their addresses, so expanded or overlapping rows are not for them.
static bool var_mfma_ok(const VitkAttnVar* a, bool bwd) {
  if (a->Dh % 8 || a->algo == 1 || a->B * a->Lq * a->Lk == 0) return false;   // (the rules below divide by their counts)
  const int es = a->dtype == VITK_BF16 ? 2 : 4;
  for (int i = 0; i < (bwd ? 24 : 12); i++)
    if (a->st[i] * es % 16 || (i % 3 == 2 && a->st[i] < a->Dh)) return false;
  const void* ps[] = {a->q, a->k, a->v, a->o, a->dout, a->dq, a->dk, a->dv};
  for (int i = 0; i < (bwd ? 8 : 4); i++)
    if ((uintptr_t)ps[i] & 15) return false;
  const int64_t lim = (1ll << 30) / es;   // elements
  if ((a->Lq + 256) * a->st[2] >= lim || (a->Lk + 256) * a->st[5] >= lim || (a->Lk + 256) * a->st[8] >= lim || (a->Lq + 256) * a->st[11] >= lim) return false;
  return !bwd || (a->Lq + 256) * a->st[14] < lim;
}
// Few queries: the kernels that read K and V once, with 32 keys per wave
static bool var_few(const VitkAttnVar* a) { return a->dtype == VITK_BF16 && a->Lq <= 32 && !(a->drop_p > 0.f); }
// Waves per workgroup, 32 query rows each: 4, or 2 where 64 rows hold all queries.
static int var_nw(const VitkAttnVar* a) { return a->Lq <= 64 && !(a->drop_p > 0.f) ? 2 : 4; }
// Workgroups that share the keys of a (sample, head) in the forward pass: 1 where the query blocks alone fill the chip
// (256 CUs, two workgroups each), otherwise as many as do, each with at least four 64-key tiles.
static int var_fwd_splits(const VitkAttnVar* a) {
  if (a->dtype == VITK_F32) {   // one wave of 32 queries per workgroup, 32-key tiles
    const int64_t waves = a->B * a->H * ceil_div(a->Lq, 32), tiles = ceil_div(a->Lk, 32);
    if (waves >= 1024 || tiles < 4) return 1;
    int64_t n = ceil_div(1024, waves);
    if (n > tiles / 2) n = tiles / 2;
    return (int)(n < 64 ? n : 64);
  }
  if (var_few(a)) {   // shares are waves, up to 4 of a workgroup: four rounds of the four waves a CU holds
    const int64_t kw = 4 / var_few_heads(a->H);
    int64_t n = 4096 / (a->B * a->H), most = ceil_div(a->Lk, 32) / 4;
    if (n > most) n = most;
    if (n > 64) n = 64;
    return (int)(ceil_div(n < 1 ? 1 : n, kw) * kw);
  }
  if (a->drop_p > 0.f) return 1;
  const int64_t blocks = a->B * a->H * ceil_div(a->Lq, 32 * var_nw(a)), tiles = ceil_div(a->Lk, 64);
  if (blocks >= 512 || tiles < 8) return 1;
  int64_t n = ceil_div(768, blocks);
  if (n > tiles / 4) n = tiles / 4;
  return (int)(n < 64 ? n : 64);
}
// Shares of the samples in the bias gradient: float32 enough workgroups to fill the chip twice; bf16, where a CU holds two (one
// with heads beyond 96), as many as run at once at most (the next would run after the others).
static int var_dbias_splits(const VitkAttnVar* a) {
  const bool f32 = a->dtype == VITK_F32;
  const int rows = f32 ? 32 : 64;   // queries of a workgroup
  const int64_t blocks = a->H * ceil_div(a->Lq, rows) * ceil_div(a->Lk, 128);
  int64_t n = f32 ? ceil_div(512, blocks) : (a->Dh <= 96 ? 512 : 256) / blocks;
  if (n > a->B) n = a->B;
  return (int)(n < 1 ? 1 : n);
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
struct VarWs { size_t delta, nl, bias_s, bias_t, dbias, pieces, part, pstat, total; int splits; };
static VarWs var_ws(const VitkAttnVar* a, bool bwd) {
  VarWs w = {};
  w.splits = 1;
  const bool mfma = var_mfma_ok(a, bwd);
  const size_t rows = (size_t)(a->B * a->H * a->Lq);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t here = at; at += up256(n); return here; };
  if (mfma && a->bias_table && a->dtype == VITK_BF16) {
    w.bias_s = take((size_t)a->H * ceil_div(a->Lq, 32) * ceil_div(a->Lk, 64) * 2 * 2048);
    if (bwd) w.bias_t = take((size_t)a->H * ceil_div(a->Lk, 32) * ceil_div(a->Lq, 64) * 2 * 2048);
  }
  if (!bwd) {
    w.splits = mfma ? var_fwd_splits(a) : 1;
    if (w.splits > 1) { w.part = take(w.splits * rows * a->Dh * 4); w.pstat = take(w.splits * rows * 8); }
  } else {
    w.delta = take(rows * 4);
    w.nl = take(rows * 4);
    if (mfma && var_few(a)) {
      w.part = take((size_t)ceil_div(a->Lk, 128) * rows * a->Dh * 4);
      if (a->dbias_table) w.pstat = take((size_t)ceil_div(a->Lk, 128) * rows * 8);
    }
    if (a->dbias_table) {
      w.splits = mfma ? var_dbias_splits(a) : 1;
      w.dbias = take((size_t)w.splits * a->H * a->Lq * a->Lk * 4);
      w.pieces = take((size_t)a->H * a->num_pieces * 4);
    }
  }
  w.total = at;
  return w;
}
extern "C" size_t vitk_attn_var_workspace_bytes(const VitkAttnVar* a, int bwd) {
  if (!a || var_validate(a, bwd != 0)) return 0;
  const VitkAttnVar n = var_normal(a);
  return var_ws(&n, bwd != 0).total;
}
#define VAR_T(T, ...) do { if (a->dtype == VITK_F32) { typedef float T; __VA_ARGS__; } else { typedef bf16 T; __VA_ARGS__; } } while (0)

extern "C" int vitk_attn_var_fwd(const VitkAttnVar* desc, void* stream) {
  if (int rc = var_validate(desc, false)) return rc;
  const VitkAttnVar normal = var_normal(desc), *a = &normal;
  if (a->B == 0 || a->Lq == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  VarP p = make_varp(a);
  const VarWs w = var_ws(a, false);
  VITK_REQUIRE(w.total == 0 || (a->workspace && a->workspace_bytes >= (int64_t)w.total), "attn_var_fwd: workspace too small");
  const bool mfma = var_mfma_ok(a, false);
  VITK_REQUIRE(a->algo != 2 || mfma, "attn_var_fwd: the matrix-unit kernels cannot take this problem (dtype, alignment, head size)");
  if (mfma) {
    char* ws = (char*)a->workspace;
    p.splits = w.splits;
    p.part = (float*)(ws + w.part);
    p.pstat = (float*)(ws + w.pstat);
    if (a->dtype == VITK_F32) {
      f32_launch_fwd(p, st);
      if (p.splits > 1) var_launch_combine(p, true, st);
    } else {
      if (a->bias_table) {
        p.bias_s = (const bf16*)(ws + w.bias_s);
        var_launch_expand(p, false, st);
      }
      if (var_few(a)) var_launch_few_fwd(p, a->bias_table != nullptr, st);
      else var_launch_fwd(p, a->bias_table != nullptr, var_nw(a), st);
    }
  } else {
    dim3 grid((unsigned)ceil_div(a->Lq, 64), (unsigned)a->H, (unsigned)a->B);
    const size_t lds = (size_t)2 * VT * a->Dh * sizeof(float);
    VAR_T(T, hipLaunchKernelGGL((var_fwd_simple_k<T>), grid, dim3(256), lds, st, p));
  }
  VITK_LAUNCH_CHECK("attn_var_fwd");
  return 0;
}

extern "C" int vitk_attn_var_bwd(const VitkAttnVar* desc, void* stream) {
  if (int rc = var_validate(desc, true)) return rc;
  const VitkAttnVar normal = var_normal(desc), *a = &normal;
  if (a->B * (a->Lq + a->Lk) == 0 && !a->dbias_table) return 0;
  hipStream_t st = (hipStream_t)stream;
  VarP p = make_varp(a);
  const VarWs w = var_ws(a, true);
  VITK_REQUIRE(w.total == 0 || (a->workspace && a->workspace_bytes >= (int64_t)w.total), "attn_var_bwd: workspace too small");
  char* ws = (char*)a->workspace;
  p.delta = (float*)(ws + w.delta);
  p.nl = (float*)(ws + w.nl);
  p.dbias = (float*)(ws + w.dbias);
  p.part = (float*)(ws + w.part);
  p.splits = w.splits;
  const int64_t rows = a->B * a->H * a->Lq;
  const bool mfma = var_mfma_ok(a, true) && rows > 0, bias = a->bias_table != nullptr;
  VITK_REQUIRE(a->algo != 2 || mfma, "attn_var_bwd: the matrix-unit kernels cannot take this problem (dtype, alignment, head size)");
  const size_t lds = (size_t)2 * VT * a->Dh * sizeof(float);
  const int64_t pairs = a->Lq * a->Lk;
  if (mfma && a->dtype == VITK_F32) {
    f32_launch_bwd(p, st);   // dQ and delta, then dK and dV
    if (a->dbias_table) f32_launch_dbias(p, st);
  } else if (mfma) {
    if (bias) {
      p.bias_s = (const bf16*)(ws + w.bias_s);
      p.bias_t = (const bf16*)(ws + w.bias_t);
      var_launch_expand(p, true, st);
    }
    if (var_few(a)) {
      if (a->dbias_table) p.pstat = (float*)(ws + w.pstat);
      var_launch_few_bwd(p, bias, st);
    } else {
      var_launch_dq(p, bias, st);     // writes delta
      var_launch_dkdv(p, bias, st);   // reads it
    }
    if (a->dbias_table) var_launch_dbias(p, st);
  } else {
    if (rows > 0) {
      VAR_T(T, hipLaunchKernelGGL((var_delta_k<T>), dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, st, p));
      VAR_T(T, hipLaunchKernelGGL((var_dq_simple_k<T>), dim3((unsigned)ceil_div(a->Lq, 64), (unsigned)a->H, (unsigned)a->B), dim3(256), lds, st, p));
    }
    if (a->B * a->Lk > 0)
      VAR_T(T, hipLaunchKernelGGL((var_dkdv_simple_k<T>), dim3((unsigned)ceil_div(a->Lk, 64), (unsigned)a->H, (unsigned)a->B), dim3(256), lds + 512, st, p));
    if (a->dbias_table && pairs > 0)
      VAR_T(T, hipLaunchKernelGGL((var_dbias_simple_k<T>), dim3((unsigned)ceil_div(pairs, 256), (unsigned)a->H), dim3(256), 0, st, p));
  }
  if (a->dbias_table) {
    float* part = (float*)(ws + w.pieces);
    if (a->num_pieces > 0)
      hipLaunchKernelGGL(var_piece_sum_k, dim3(xcd_grid(ceil_div(a->num_pieces, 4) * ceil_div(a->H, 4))), dim3(256), 0, st, p.dbias, a->order, a->piece, part, pairs, (int)a->H, (int)a->num_pieces, w.splits);
    const dim3 bgrid((unsigned)a->num_buckets, (unsigned)a->H);
    if (a->dbias_dtype == VITK_F32)
      hipLaunchKernelGGL((var_bucket_sum_k<float>), bgrid, dim3(256), 0, st, part, a->bucket_piece, (float*)a->dbias_table, (int)a->H, (int)a->num_pieces);
    else
      hipLaunchKernelGGL((var_bucket_sum_k<bf16>), bgrid, dim3(256), 0, st, part, a->bucket_piece, (bf16*)a->dbias_table, (int)a->H, (int)a->num_pieces);
  }
  VITK_LAUNCH_CHECK("attn_var_bwd");
  return 0;
}
