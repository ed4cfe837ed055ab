// Per-head normalisation of q and k with the position rotation in the same pass, forward and backward.
//
//   xhat = (x - mean) * rstd   (RMSNorm: mean = 0),   n = xhat * w (+ b)          over the Dh values of a head
//   y    = n * cos + rotate_half(n) * sin             for the rows behind the prefix, n elsewhere
// Backward, with g = the gradient of y:
//   dn   = g * cos + rotate_half^T(g * sin),  dw = sum dn * xhat,  db = sum dn
//   dx   = rstd * (u - xhat * mean(u * xhat) - mean(u)),  u = dn * w   (RMSNorm without the last mean)
// The statistics are taken again from x in the backward: the head is in registers anyway, and nothing is kept between the
// two passes.  A row of a head lies on a group of G lanes; every lane holds V values of the first half of the head and the
// V values Dh / 2 further on, so that the rotation stays inside the lane.  A wave walks the heads of one token at a time
// with the token's sines and cosines in registers.  Bound by HBM: x in, y out (forward), g and x in, dx out (backward).
#include "common.h"

struct QkSec {        // one section: q or k
  const void *x, *g;  // input; gradient of the output (backward)
  void* y;            // output (forward) or gradient of x (backward)
  const void *w, *b;
  void *dw, *db;
  const float* table;   // [2, (B,) L - prefix, Dh] or NULL
  int64_t x_sb, x_ss, x_sh, g_sb, g_ss, g_sh, y_sb, y_ss, y_sh;
  int64_t tok_stride;   // table elements between samples (0: shared)
  int64_t cos_off;      // elements from the sines to the cosines
  int L, H, prefix;
};
struct QkP {
  QkSec s[2];
  float* partial;   // [2 sections][2: dw, db][gridDim.x][Dh]
  int B, Dh;
  float eps;
  int ln, round_norm, emu, want_dw;
};

template <int G> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <class T, int V> __device__ __forceinline__ void load_n(float (&r)[V], const T* p) {
  VecN<T, V> t;
  t.load(p);
#pragma unroll
  for (int i = 0; i < V; i++) r[i] = t.v[i];
}
template <class T, int V> __device__ __forceinline__ void store_n(T* p, const float (&r)[V]) {
  VecN<T, V> t;
#pragma unroll
  for (int i = 0; i < V; i++) t.v[i] = r[i];
  t.store(p);
}
template <class TW> __device__ __forceinline__ float opt_load(const void* p, int i, float dflt) {
  return p ? to_f<TW>(((const TW*)p)[i]) : dflt;
}
template <int V> __device__ __forceinline__ void load_table(float (&r)[V], const float* p) {
#pragma unroll
  for (int i = 0; i < V; i += 4) *(float4*)(r + i) = *(const float4*)(p + i);
}

template <class T, class TW, int V, int G, bool BWD>
__global__ __launch_bounds__(256) void qk_norm_rope_k(QkP p) {
  constexpr int HPW = 64 / G;   // heads a wave handles at a time
  const QkSec& s = p.s[blockIdx.y];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane % G, hl = lane / G, half = p.Dh >> 1;
  const bool on = j * V < half;
  const int d0 = on ? j * V : 0, d1 = d0 + half;
  const float inv_n = 1.f / (float)p.Dh;
  float w0[V], w1[V], b0[V], b1[V], gw0[V], gw1[V], gb0[V], gb1[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    w0[i] = to_f<TW>(((const TW*)s.w)[d0 + i]); w1[i] = to_f<TW>(((const TW*)s.w)[d1 + i]);
    b0[i] = BWD ? 0.f : opt_load<TW>(s.b, d0 + i, 0.f); b1[i] = BWD ? 0.f : opt_load<TW>(s.b, d1 + i, 0.f);
    gw0[i] = gw1[i] = gb0[i] = gb1[i] = 0.f;
  }
  const int64_t tokens = (int64_t)p.B * s.L;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wid; t < tokens; t += (int64_t)gridDim.x * 4) {
    const int64_t b = t / s.L;
    const int l = (int)(t - b * s.L);
    const bool rot = s.table != nullptr && l >= s.prefix;
    float s0[V], s1[V], c0[V], c1[V];
    if (rot) {
      const float* tp = s.table + b * s.tok_stride + (int64_t)(l - s.prefix) * p.Dh;
      load_table<V>(s0, tp + d0); load_table<V>(s1, tp + d1);
      load_table<V>(c0, tp + s.cos_off + d0); load_table<V>(c1, tp + s.cos_off + d1);
    }
    const T* xt = (const T*)s.x + b * s.x_sb + (int64_t)l * s.x_ss;
    const T* gt = BWD ? (const T*)s.g + b * s.g_sb + (int64_t)l * s.g_ss : nullptr;
    T* yt = (T*)s.y + b * s.y_sb + (int64_t)l * s.y_ss;
    for (int h0 = 0; h0 < s.H; h0 += HPW) {
      const int h = h0 + hl;
      const bool live = on && h < s.H;
      float x0[V], x1[V], g0[V], g1[V];
      if (live) {
        load_n<T, V>(x0, xt + h * s.x_sh + d0); load_n<T, V>(x1, xt + h * s.x_sh + d1);
        if (BWD) { load_n<T, V>(g0, gt + h * s.g_sh + d0); load_n<T, V>(g1, gt + h * s.g_sh + d1); }
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) { x0[i] = x1[i] = 0.f; g0[i] = g1[i] = 0.f; }
      }
      if (p.ln) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) m += x0[i] + x1[i];
        m = group_sum<G>(m) * inv_n;
#pragma unroll
        for (int i = 0; i < V; i++) { x0[i] -= m; x1[i] -= m; }
      }
      float q = 0.f;
      if (live) {
#pragma unroll
        for (int i = 0; i < V; i++) { q = fmaf(x0[i], x0[i], q); q = fmaf(x1[i], x1[i], q); }
      }
      const float rstd = rsqrtf(group_sum<G>(q) * inv_n + p.eps);
      if (!BWD) {
        float y0[V], y1[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
          float n0 = norm_apply(x0[i], rstd, w0[i], b0[i], s.b != nullptr), n1 = norm_apply(x1[i], rstd, w1[i], b1[i], s.b != nullptr);
          if (p.round_norm) { n0 = round_as<T>(n0); n1 = round_as<T>(n1); }
          y0[i] = rot ? rope_mix(n0, c0[i], -n1, s0[i], p.emu) : n0;
          y1[i] = rot ? rope_mix(n1, c1[i], n0, s1[i], p.emu) : n1;
        }
        if (live) { store_n<T, V>(yt + h * s.y_sh + d0, y0); store_n<T, V>(yt + h * s.y_sh + d1, y1); }
      } else {
        float a = 0.f, c = 0.f;   // sums of u * xhat and of u
#pragma unroll
        for (int i = 0; i < V; i++) {
          float n0 = rot ? rope_mix(g0[i], c0[i], g1[i], s1[i], p.emu) : g0[i];
          float n1 = rot ? rope_mix(g1[i], c1[i], -g0[i], s0[i], p.emu) : g1[i];
          if (p.round_norm && rot) { n0 = round_as<T>(n0); n1 = round_as<T>(n1); }
          x0[i] *= rstd; x1[i] *= rstd;
          if (live) {
            gw0[i] = fmaf(n0, x0[i], gw0[i]); gw1[i] = fmaf(n1, x1[i], gw1[i]);
            gb0[i] += n0; gb1[i] += n1;
            g0[i] = n0 * w0[i]; g1[i] = n1 * w1[i];
            a = fmaf(g0[i], x0[i], a); a = fmaf(g1[i], x1[i], a);
            c += g0[i] + g1[i];
          }
        }
        a = group_sum<G>(a) * inv_n;
        c = p.ln ? group_sum<G>(c) * inv_n : 0.f;
        if (live) {
#pragma unroll
          for (int i = 0; i < V; i++) {
            g0[i] = (g0[i] - c - x0[i] * a) * rstd;
            g1[i] = (g1[i] - c - x1[i] * a) * rstd;
          }
          store_n<T, V>(yt + h * s.y_sh + d0, g0); store_n<T, V>(yt + h * s.y_sh + d1, g1);
        }
      }
    }
  }
  if (BWD && p.want_dw) {   // sums of the workgroup: groups of a wave by shuffles, waves through LDS, always in this order
    __shared__ float red[4][2][128];
#pragma unroll
    for (int i = 0; i < V; i++) {
#pragma unroll
      for (int o = G; o < 64; o <<= 1) {
        gw0[i] += __shfl_xor(gw0[i], o, 64); gw1[i] += __shfl_xor(gw1[i], o, 64);
        gb0[i] += __shfl_xor(gb0[i], o, 64); gb1[i] += __shfl_xor(gb1[i], o, 64);
      }
      if (on && hl == 0) {
        red[wid][0][d0 + i] = gw0[i]; red[wid][0][d1 + i] = gw1[i];
        red[wid][1][d0 + i] = gb0[i]; red[wid][1][d1 + i] = gb1[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.Dh; i += 256) {
      const int which = i >= p.Dh, d = i - which * p.Dh;
      p.partial[((int64_t)(blockIdx.y * 2 + which) * gridDim.x + blockIdx.x) * p.Dh + d] =
          (red[0][which][d] + red[1][which][d]) + (red[2][which][d] + red[3][which][d]);
    }
  }
}

// dw / db of a section from the per-workgroup sums: block = (section, dw or db); 8 row groups x 128 columns
template <class TW> __global__ __launch_bounds__(1024) void qk_norm_rope_reduce_k(QkP p, int nblk) {
  __shared__ float red[8][128];
  const QkSec& s = p.s[blockIdx.x >> 1];
  TW* out = (TW*)((blockIdx.x & 1) ? s.db : s.dw);
  const int d = threadIdx.x & 127, r = threadIdx.x >> 7;
  const float* src = p.partial + (int64_t)blockIdx.x * nblk * p.Dh;
  float a = 0.f;
  if (out && d < p.Dh)
    for (int i = r; i < nblk; i += 8) a += src[(int64_t)i * p.Dh + d];
  red[r][d] = a;
  __syncthreads();
  if (out && r == 0 && d < p.Dh) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) t += red[i][d];
    out[d] = from_f<TW>(t);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int qk_blocks(const VitkQkNormRope* a, bool bwd) {
  int64_t tok = a->sec[0].L * a->B;
  if (a->sec[1].w && a->sec[1].L * a->B > tok) tok = a->sec[1].L * a->B;
  const int64_t want = ceil_div(tok, 4);
  const int64_t cap = bwd ? 1024 : 16384;   // backward: one partial row per workgroup
  return (int)(want < cap ? (want < 1 ? 1 : want) : cap);
}
extern "C" size_t vitk_qk_norm_rope_workspace_bytes(const VitkQkNormRope* a) {
  if (!a) return 0;
  return (size_t)4 * qk_blocks(a, true) * a->Dh * sizeof(float);
}

template <bool BWD> static int qk_norm_rope_run(const VitkQkNormRope* a, hipStream_t st) {
  const char* name = BWD ? "qk_norm_rope_bwd" : "qk_norm_rope_fwd";
  VITK_REQUIRE(a, "%s: null descriptor", name);
  VITK_REQUIRE(a->dtype == VITK_F32 || a->dtype == VITK_BF16, "%s: bad dtype", name);
  VITK_REQUIRE(a->w_dtype == VITK_F32 || a->w_dtype == VITK_BF16, "%s: bad weight dtype", name);
  VITK_REQUIRE(a->Dh >= 8 && a->Dh <= 128 && a->Dh % 8 == 0, "%s: head_dim=%lld must be a multiple of 8, at most 128", name, (long long)a->Dh);
  VITK_REQUIRE(a->B >= 0 && a->B < (1ll << 31), "%s: bad batch", name);
  QkP p;
  p.B = (int)a->B; p.Dh = (int)a->Dh; p.eps = a->eps; p.ln = a->is_layernorm; p.round_norm = a->round_norm; p.emu = a->emulate_bf16;
  p.partial = (float*)a->workspace;
  const int es = a->dtype == VITK_BF16 ? 2 : 4;
  bool v8 = a->dtype == VITK_BF16 && a->Dh % 16 == 0;
  bool want = false;
  int nsec = 0;
  for (int i = 0; i < 2; i++) {
    const VitkQkSection& q = a->sec[i];
    QkSec& s = p.s[i];
    if (i == 1 && !q.w) { s = p.s[0]; break; }
    nsec = i + 1;
    VITK_REQUIRE(q.w && (a->B * q.L == 0 || (q.x && q.y && (!BWD || q.g))), "%s: null pointer", name);
    VITK_REQUIRE(q.L >= 0 && q.H > 0 && q.L < (1ll << 31) && q.H < (1ll << 31), "%s: bad shape L=%lld H=%lld", name, (long long)q.L, (long long)q.H);
    VITK_REQUIRE(q.prefix >= 0 && q.prefix <= q.L, "%s: prefix=%lld outside [0, %lld]", name, (long long)q.prefix, (long long)q.L);
    VITK_REQUIRE(!q.table || ((uintptr_t)q.table & 15) == 0, "%s: the rotation table must be 16-byte aligned", name);
    const int64_t st_[] = {q.x_sb, q.x_ss, q.x_sh, q.y_sb, q.y_ss, q.y_sh, BWD ? q.g_sb : 0, BWD ? q.g_ss : 0, BWD ? q.g_sh : 0};
    const void* ps[] = {q.x, q.y, BWD ? q.g : q.x};
    for (int64_t x : st_) {
      VITK_REQUIRE(x % 4 == 0, "%s: strides must be multiples of 4 elements", name);
      if (x % 8) v8 = false;
    }
    for (const void* x : ps) {
      VITK_REQUIRE((uintptr_t)x % (4 * es) == 0, "%s: pointers must be aligned to 4 elements", name);
      if ((uintptr_t)x % 16) v8 = false;
    }
    s.x = q.x; s.g = q.g; s.y = q.y; s.w = q.w; s.b = q.b; s.dw = q.dw; s.db = q.db; s.table = q.table;
    s.x_sb = q.x_sb; s.x_ss = q.x_ss; s.x_sh = q.x_sh; s.g_sb = q.g_sb; s.g_ss = q.g_ss; s.g_sh = q.g_sh;
    s.y_sb = q.y_sb; s.y_ss = q.y_ss; s.y_sh = q.y_sh;
    const int64_t n = q.L - q.prefix;
    s.tok_stride = q.per_sample ? n * a->Dh : 0;
    s.cos_off = (q.per_sample ? a->B : 1) * n * a->Dh;
    s.L = (int)q.L; s.H = (int)q.H; s.prefix = (int)q.prefix;
    if (BWD && (q.dw || q.db)) want = true;
  }
  p.want_dw = want;
  VITK_REQUIRE(!want || a->workspace, "%s: workspace required for the weight gradients", name);
  const int nb = qk_blocks(a, BWD);
  const dim3 grid((unsigned)nb, (unsigned)nsec), block(256);
  const int lanes = (int)a->Dh / (v8 ? 16 : 8);   // lanes that hold a row
#define QK_GO(T, TW, V, G) hipLaunchKernelGGL((qk_norm_rope_k<T, TW, V, G, BWD>), grid, block, 0, st, p)
#define QK_G(T, TW, V) do { if (lanes <= 2) QK_GO(T, TW, V, 2); else if (lanes <= 4) QK_GO(T, TW, V, 4); else if (lanes <= 8) QK_GO(T, TW, V, 8); else QK_GO(T, TW, V, 16); } while (0)
#define QK_W(T, V) do { if (a->w_dtype == VITK_F32) QK_G(T, float, V); else QK_G(T, bf16, V); } while (0)
  if (a->dtype == VITK_F32) QK_W(float, 4);
  else if (v8) QK_W(bf16, 8);
  else QK_W(bf16, 4);
  VITK_LAUNCH_CHECK(name);
  if (BWD && want) {
    if (a->w_dtype == VITK_F32) hipLaunchKernelGGL((qk_norm_rope_reduce_k<float>), dim3(2 * nsec), dim3(1024), 0, st, p, nb);
    else hipLaunchKernelGGL((qk_norm_rope_reduce_k<bf16>), dim3(2 * nsec), dim3(1024), 0, st, p, nb);
    VITK_LAUNCH_CHECK(name);
  }
  return 0;
}
extern "C" int vitk_qk_norm_rope_fwd(const VitkQkNormRope* a, void* stream) { return qk_norm_rope_run<false>(a, (hipStream_t)stream); }
extern "C" int vitk_qk_norm_rope_bwd(const VitkQkNormRope* a, void* stream) { return qk_norm_rope_run<true>(a, (hipStream_t)stream); }
