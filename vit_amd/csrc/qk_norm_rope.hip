// Per-head normalisation of q and k with the position rotation in the same pass, forward and backward.
//
//   xhat = (x - mean) * rstd   (RMSNorm: mean = 0),   n = xhat * w (+ b)          over the Dh values of a head
//   y    = n * cos + rotate_half(n) * sin             for the rows behind the prefix, n elsewhere
// Backward, with g = the gradient of y:
//   dn   = g * cos + rotate_half^T(g * sin),  dw = sum dn * xhat,  db = sum dn
//   dx   = rstd * (u - xhat * mean(u * xhat) - mean(u)),  u = dn * w   (RMSNorm without the last mean)
// The statistics are taken again from x in the backward: the head is in registers anyway, and nothing is kept between the
// two passes.  A lane holds 8 consecutive values of a head (16 bytes in bf16), a wave as many whole rows as fit, so that its
// loads and stores are one contiguous run where the rows are; the other half of the head that the rotation needs and the
// row sums go through LDS.  Positions come before samples in a wave's run: their sines and cosines stay in registers.
// Bound by HBM: x in, y out (forward), g and x in, dx out (backward; its vector instructions come close).  Measured in bf16:
// ViT-H/14 at 224 px, 64 samples, 16 + 16 heads of 80: forward 35 us (4.7 TB/s), backward 58 us (4.3 TB/s); ViT-g/14 at 1024 px, 8
// samples, heads of 88: 102 us (4.7 TB/s) and 180 us (4.0 TB/s), where a copy reaches 5.1 TB/s; the weight gradients' partial
// sums take 4-5 us more.  One token of 12 + 12 heads takes 4 us, a launch.
// Instances: head sizes 32, 64, 96, 128 and those of the larger ViTs (80, 88) know their lanes per row when compiled, which folds
// the row sums; the others, and float32 rows with bf16 weights, take the same code with the count in a register.  64 samples x
// 257 tokens, 16 + 16 heads, forward / training, instance against general form: heads of 32 in bf16 20 / 42 against 22 / 48 us,
// 64: 29 / 64 against 32 / 72, 80: 37 / 93 against 39 / 101, 88: 40 / 113 against 42 / 120, 96: 43 / 120 against 44 / 126, 128: 58 / 139 against 62 / 152; float32
// 64: 60 / 136 against 69 / 149, 96: no difference, 128: 124 / 272 against 151 / 297.  Sizes between them stay near their
// neighbours' bandwidth without an instance (72: 36 / 88, 104: 49 / 143, 120: 60 / 155 us).
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

// Eight consecutive values of a head as they lie in memory
template <class T> struct Raw8;
template <> struct Raw8<bf16> { uint4 a; };
template <> struct Raw8<float> { uint4 a, b; };
template <class T> __device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
  r.a = *(const uint4*)p;
  if constexpr (sizeof(T) == 4) r.b = *(const uint4*)(p + 4);
  return r;
}
template <class T> __device__ __forceinline__ void unpack8(float (&v)[8], const Raw8<T>& r) {
  T e[8];
  __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = to_f<T>(e[i]);
}
template <class T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; i++) e[i] = from_f<T>(v[i]);
  Raw8<T> r;
  __builtin_memcpy(&r, e, sizeof(r));
  *(uint4*)p = r.a;
  if constexpr (sizeof(T) == 4) *(uint4*)(p + 4) = r.b;
}

// Lanes of a wave hand values to each other through LDS, which a wave's accesses pass in order; this keeps the compiler from
// moving one lane's read ahead of another's write.  No instruction comes of it.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// NL = lanes of a row, Dh / 8 (0: taken from the descriptor).  SEP: the roundings of separate passes are wanted (round_norm,
// emulate_bf16); otherwise products are fused into the sums.
template <class T, class TW, int NL, bool SEP, bool BWD>
__global__ __launch_bounds__(256, 4) void qk_norm_rope_k(QkP p) {
  constexpr int EX = 64 * 8, SUMS = 64 * 4;   // a wave's values handed to the other half of a head; partial sums (rows x 16)
  __shared__ __attribute__((aligned(16))) float shared[4][EX + SUMS];
  const QkSec s = blockIdx.y == 0 ? p.s[0] : p.s[1];
  const int H = s.H;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nl = NL ? NL : p.Dh >> 3, Dh = nl * 8, rpw = nl == 3 ? 16 : 64 / nl, rr = lane / nl, j = lane - rr * nl, d0 = 8 * j;
  const bool on = rr < rpw;
  float* ex = shared[wid] + (on ? rr : 0) * Dh;
  float* sums = shared[wid] + EX + (on && rpw <= 16 ? rr : 0) * 16;
  // the lane's two quads and where their partners lie, half a head (nl quads) away; a first-half quad takes -sin
  const int qa = 2 * j, qb = 2 * j + 1;
  const int pa = 4 * (qa < nl ? qa + nl : qa - nl), pb = 4 * (qb < nl ? qb + nl : qb - nl);
  const float sga = qa < nl ? -1.f : 1.f, sgb = qb < nl ? -1.f : 1.f;
  const float inv_n = 1.f / (float)Dh;
  const bool has_b = !BWD && s.b != nullptr, has_table = s.table != nullptr;
  float w[8], bias[8], gw[8], gb[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    w[i] = on ? to_f<TW>(((const TW*)s.w)[d0 + i]) : 0.f;
    bias[i] = has_b && on ? to_f<TW>(((const TW*)s.b)[d0 + i]) : 0.f;
    gw[i] = gb[i] = 0.f;
  }
  // Sum over the lanes of a row, the same value in all of them: by shuffles where they are a power of two, else through LDS,
  // in the lanes' order
  auto row_sum = [&](float v) {
    if (NL == 4 || NL == 8 || NL == 16) {
#pragma unroll
      for (int o = NL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
      return v;
    }
    if (nl <= 2) return nl == 1 ? v : v + __shfl_xor(v, 1, 64);
    wave_order();
    if (on) sums[j] = v;   // at most 16 rows
    wave_order();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (4 * i < nl) {
        const float4 q = *(const float4*)(sums + 4 * i);
        t += 4 * i + 3 < nl ? (q.x + q.y) + (q.z + q.w) : 4 * i + 2 < nl ? q.x + q.y + q.z : 4 * i + 1 < nl ? q.x + q.y : q.x;
      }
    }
    return t;
  };
  // Rows in the order position, sample, head: a wave takes a run of them, rpw at a time, so that all its lanes but those that
  // no row fits in are busy (16 heads of 88 taken token by token: 5 + 5 + 5 + 1 of 5).  A row's place moves by a fixed step,
  // corrected where the heads or the samples wrap; its sines and cosines stay until the position changes.
  const int64_t rows = (int64_t)p.B * s.L * H, nw = (int64_t)gridDim.x * 4;
  const int64_t run = ((rows + nw - 1) / nw + rpw - 1) / rpw * rpw;
  const int64_t r0 = run * ((int64_t)blockIdx.x * 4 + wid), r1 = r0 + run < rows ? r0 + run : rows;
  if (r0 < r1) {
    const int B = p.B, step_t = rpw / H, sh = rpw - step_t * H, sl = step_t / B, sb = step_t - sl * B;   // rpw rows further
    const int64_t xs = sl * s.x_ss + sb * s.x_sb + sh * s.x_sh, ys = sl * s.y_ss + sb * s.y_sb + sh * s.y_sh;
    const int64_t xb = s.x_sb - H * s.x_sh, yb = s.y_sb - H * s.y_sh, xl = s.x_ss - B * s.x_sb, yl = s.y_ss - B * s.y_sb;
    const int64_t gs = BWD ? sl * s.g_ss + sb * s.g_sb + sh * s.g_sh : 0, gb_ = BWD ? s.g_sb - H * s.g_sh : 0, gl = BWD ? s.g_ss - B * s.g_sb : 0;
    const int64_t first = r0 + rr;
    int64_t t = first / H;
    int h = (int)(first - t * H), l = (int)(t / B), b = (int)(t - (int64_t)l * B), table_l = -1;
    const T* xp = (const T*)s.x + b * s.x_sb + l * s.x_ss + h * s.x_sh + d0;
    const T* gp = BWD ? (const T*)s.g + b * s.g_sb + l * s.g_ss + h * s.g_sh + d0 : nullptr;
    T* yp = (T*)s.y + b * s.y_sb + l * s.y_ss + h * s.y_sh + d0;
    const float* table = s.table;
    const int64_t tok_stride = s.tok_stride, cos_off = s.cos_off;
    const int prefix = s.prefix;
    const bool ln = p.ln;
    const float eps = p.eps;
    int left = on ? (int)min((int64_t)INT32_MAX, r1 - first) : 0;   // rows from the lane's on: none left where not above 0
    auto fetch = [&](Raw8<T>& xr, Raw8<T>& gr) {
      if (left > 0) {
        xr = load8<T>(xp);
        if (BWD) gr = load8<T>(gp);
      }
    };
    float sn[8], cs[8];
#pragma unroll
    for (int i = 0; i < 8; i++) { sn[i] = 0.f; cs[i] = 1.f; }
    Raw8<T> xr = {}, gr = {};
    fetch(xr, gr);
    for (int64_t n = r1 - r0; n > 0; n -= rpw) {
      const int lc = l, bc = b;
      const bool live = left > 0;
      float x[8], g[8];
      unpack8<T>(x, xr);
      if (BWD) unpack8<T>(g, gr);
      T* const yc = yp;
      h += sh; b += sb; l += sl; left -= rpw;
      xp += xs; yp += ys;
      if (BWD) gp += gs;
      if (h >= H) {
        h -= H; b++;
        xp += xb; yp += yb;
        if (BWD) gp += gb_;
      }
      if (b >= B) {
        b -= B; l++;
        xp += xl; yp += yl;
        if (BWD) gp += gl;
      }
      fetch(xr, gr);   // the next rows are asked for before these are worked on
      const bool rot = has_table && lc >= prefix && live;
      if (rot && (lc != table_l || tok_stride)) {
        const float* tp = table + bc * tok_stride + (int64_t)(lc - prefix) * Dh + (on ? d0 : 0);
        *(float4*)sn = *(const float4*)tp; *(float4*)(sn + 4) = *(const float4*)(tp + 4);
        *(float4*)cs = *(const float4*)(tp + cos_off); *(float4*)(cs + 4) = *(const float4*)(tp + cos_off + 4);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (!BWD) sn[i] *= i < 4 ? sga : sgb;   // the sign of rotate_half goes with the sine
        table_l = lc;
      }
      if (ln) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) m += x[i];
        m = row_sum(m) * inv_n;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] -= m;
      }
      float q = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) q = fmaf(x[i], x[i], q);
      const float rstd = __builtin_amdgcn_rsqf(row_sum(q) * inv_n + eps);   // 1 ulp
      if (!BWD) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          y[i] = SEP ? norm_apply(x[i], rstd, w[i], bias[i], has_b) : fmaf(x[i] * rstd, w[i], bias[i]);
          if (SEP && p.round_norm) y[i] = round_as<T>(y[i]);
        }
        if (rot) {
          wave_order();
          if (on) {
            *(float4*)(ex + d0) = make_float4(y[0], y[1], y[2], y[3]);
            *(float4*)(ex + d0 + 4) = make_float4(y[4], y[5], y[6], y[7]);
          }
          wave_order();
          float o[8];
          *(float4*)o = *(const float4*)(ex + pa);
          *(float4*)(o + 4) = *(const float4*)(ex + pb);
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = SEP ? rope_mix(y[i], cs[i], o[i], sn[i], p.emu) : fmaf(y[i], cs[i], o[i] * sn[i]);
        }
        if (live) store8<T>(yc, y);
      } else {
        if (rot) {   // the transposed rotation: the partner sends g sin
          float t[8], o[8];
#pragma unroll
          for (int i = 0; i < 8; i++) t[i] = __fmul_rn(g[i], sn[i]);
          wave_order();
          if (on) {
            *(float4*)(ex + d0) = make_float4(t[0], t[1], t[2], t[3]);
            *(float4*)(ex + d0 + 4) = make_float4(t[4], t[5], t[6], t[7]);
          }
          wave_order();
          *(float4*)o = *(const float4*)(ex + pa);
          *(float4*)(o + 4) = *(const float4*)(ex + pb);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float sg = i < 4 ? sga : sgb;   // -1 in the first half, which adds its partner's product
            if (SEP) {
              float a = __fmul_rn(g[i], cs[i]), c = o[i];
              if (p.emu) { a = round_bf16(a); c = round_bf16(c); }
              g[i] = __fadd_rn(a, -sg * c);
              if (p.round_norm) g[i] = round_as<T>(g[i]);
            } else {
              g[i] = fmaf(g[i], cs[i], -sg * o[i]);
            }
          }
        }
        float a = 0.f, c = 0.f;   // sums of u * xhat and of u
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] *= rstd;
          if (live) { gw[i] = fmaf(g[i], x[i], gw[i]); gb[i] += g[i]; }
          g[i] *= w[i];
          a = fmaf(g[i], x[i], a);
          if (ln) c += g[i];
        }
        a = row_sum(a) * inv_n;
        c = ln ? row_sum(c) * inv_n : 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = (fmaf(-x[i], a, g[i]) - c) * rstd;
        if (live) store8<T>(yc, g);
      }
    }
  }
  if (BWD && p.want_dw) {   // sums of the workgroup over the rows of its waves, always in this order: dw, then db
    for (int which = 0; which < 2; which++) {
      __syncthreads();
      if (on) {
#pragma unroll
        for (int i = 0; i < 8; i++) ex[d0 + i] = which ? gb[i] : gw[i];
      }
      __syncthreads();
      for (int d = threadIdx.x; d < Dh; d += 256) {
        float t = 0.f;
        for (int v = 0; v < 4; v++)
          for (int r = 0; r < rpw; r++) t += shared[v][r * Dh + d];
        p.partial[((int64_t)(blockIdx.y * 2 + which) * gridDim.x + blockIdx.x) * Dh + d] = t;
      }
    }
  }
}

// dw / db of a section from the per-workgroup sums: a workgroup per (section, dw or db) and 8 columns; 128 row groups, their
// sums joined in a tree through LDS
template <class TW> __global__ __launch_bounds__(1024) void qk_norm_rope_reduce_k(QkP p, int nblk) {
  __shared__ float red[128][8];
  const int which = blockIdx.y, c = threadIdx.x & 7, r = threadIdx.x >> 3, d = (int)blockIdx.x * 8 + c;
  const QkSec& s = p.s[which >> 1];
  TW* out = (TW*)((which & 1) ? s.db : s.dw);
  if (!out) return;
  const float* src = p.partial + (int64_t)which * nblk * p.Dh + d;
  float a = 0.f;
  for (int i = r; i < nblk; i += 1024) {   // 8 rows in flight
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; u++) x[u] = i + 128 * u < nblk ? src[(int64_t)(i + 128 * u) * p.Dh] : 0.f;
    a += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
  }
  red[r][c] = a;
  __syncthreads();
  for (int o = 64; o > 0; o >>= 1) {
    if (r < o) red[r][c] += red[r + o][c];
    __syncthreads();
  }
  if (r == 0) out[d] = from_f<TW>(red[0][c]);
}

// ---- host ------------------------------------------------------------------------------------------------------------
static int qk_blocks(const VitkQkNormRope* a, bool bwd) {
  int64_t tok = a->sec[0].L * a->B;
  if (a->sec[1].w && a->sec[1].L * a->B > tok) tok = a->sec[1].L * a->B;
  const int64_t want = ceil_div(tok, 4);
  // As many workgroups of both sections as run at once (4 or 6 per CU), each with a longer run of rows: with twice as many, in
  // two rounds, ViT-g/14 at 1024 px takes 111 / 188 us in place of 102 / 179.  Backward: a partial sum per workgroup.
  const int64_t cap = (bwd ? 1024 : 1536) / (a->sec[1].w ? 2 : 1);
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
  const int es = a->dtype == VITK_BF16 ? 2 : 4, al = 16 / es;   // elements of 16 bytes
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
    const bool hs = q.H > 1, ls = q.L > 1, bs = a->B > 1;   // the stride of an axis of one element is never used
    const int64_t st_[] = {bs ? q.x_sb : 0, ls ? q.x_ss : 0, hs ? q.x_sh : 0, bs ? q.y_sb : 0, ls ? q.y_ss : 0, hs ? q.y_sh : 0,
                           BWD && bs ? q.g_sb : 0, BWD && ls ? q.g_ss : 0, BWD && hs ? q.g_sh : 0};
    const void* ps[] = {q.x, q.y, BWD ? q.g : q.x};
    for (int64_t x : st_) VITK_REQUIRE(x % al == 0, "%s: strides must be multiples of 16 bytes", name);
    for (const void* x : ps) VITK_REQUIRE((uintptr_t)x % 16 == 0, "%s: pointers must be 16-byte aligned", name);
    s.x = q.x; s.g = q.g; s.y = q.y; s.w = q.w; s.b = q.b; s.dw = q.dw; s.db = q.db; s.table = q.table;
    s.x_sb = st_[0]; s.x_ss = st_[1]; s.x_sh = st_[2]; s.y_sb = st_[3]; s.y_ss = st_[4]; s.y_sh = st_[5];
    s.g_sb = st_[6]; s.g_ss = st_[7]; s.g_sh = st_[8];
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
  const bool sep = a->round_norm || a->emulate_bf16;
#define QK_GO(T, TW, NL) do { \
    if (sep) hipLaunchKernelGGL((qk_norm_rope_k<T, TW, NL, true, BWD>), grid, block, 0, st, p); \
    else hipLaunchKernelGGL((qk_norm_rope_k<T, TW, NL, false, BWD>), grid, block, 0, st, p); } while (0)
#define QK_N(T, TW) do { \
    switch (a->Dh / 8) { \
      case 4: QK_GO(T, TW, 4); break; case 8: QK_GO(T, TW, 8); break; case 10: QK_GO(T, TW, 10); break; \
      case 11: QK_GO(T, TW, 11); break; case 12: QK_GO(T, TW, 12); break; case 16: QK_GO(T, TW, 16); break; \
      default: QK_GO(T, TW, 0); } } while (0)
  if (a->dtype == VITK_F32 && a->w_dtype == VITK_F32) QK_N(float, float);
  else if (a->dtype == VITK_F32) QK_GO(float, bf16, 0);
  else if (a->w_dtype == VITK_F32) QK_N(bf16, float);
  else QK_N(bf16, bf16);
  VITK_LAUNCH_CHECK(name);
  if (BWD && want) {
    const dim3 rgrid((unsigned)(a->Dh / 8), (unsigned)(2 * nsec));
    if (a->w_dtype == VITK_F32) hipLaunchKernelGGL((qk_norm_rope_reduce_k<float>), rgrid, dim3(1024), 0, st, p, nb);
    else hipLaunchKernelGGL((qk_norm_rope_reduce_k<bf16>), rgrid, dim3(1024), 0, st, p, nb);
    VITK_LAUNCH_CHECK(name);
  }
  return 0;
}
extern "C" int vitk_qk_norm_rope_fwd(const VitkQkNormRope* a, void* stream) { return qk_norm_rope_run<false>(a, (hipStream_t)stream); }
extern "C" int vitk_qk_norm_rope_bwd(const VitkQkNormRope* a, void* stream) { return qk_norm_rope_run<true>(a, (hipStream_t)stream); }
