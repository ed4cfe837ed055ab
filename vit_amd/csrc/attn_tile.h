// Building blocks of the MFMA attention kernels (bf16, v_mfma_f32_32x32x16_bf16): staging of 64-row tiles through LDS, the
// two fragment readers, the accumulator layout, stores of transposed accumulators and the workgroup order.
#pragma once
#include "common.h"

#define LOG2E 1.4426950408889634f

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

// LDS row strides (bytes) for a [64][DHP] bf16 tile.
//   ROWS: ds_read_b128 of 32 different rows at one column is conflict-free when stride/4 = 4 (mod 8) dwords
//   COLS: ds_read_b64_tr_b16 blocks of 4 rows are conflict-free when stride/4 = 16 or 48 (mod 64) dwords.
// A tile that is read both ways uses the COLS stride and stores 16-byte chunk c of row r at chunk position
// c ^ ((r >> 2) & 3): the transposing reads still find 4 rows x 64 contiguous bytes on distinct banks (the 4 rows of a
// read share (r >> 2) & 3), and the 16 rows one ds_read_b128 lane group covers now land on 16 different bank quads.
template <int DHP> struct Strides {
  static constexpr int ROWS = DHP * 2 + 16;
  static constexpr int COLS = (DHP == 96) ? 192 : DHP * 2 + 64;
};

// Operand rows come through buffer loads: a row at or beyond S starts past the descriptor's size and reads as zeros,
// a 16-byte chunk beyond the head dimension is given an offset past any size (the host keeps S * stride below 2^30 B).
constexpr uint32_t OOB_OFF = 0xC0000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const bf16* g, int64_t ss, int S, int Dh) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)g, 0, S > 0 ? (int)(((int64_t)(S - 1) * ss + Dh) * 2) : 0, 0x00020000);
}
__device__ __forceinline__ uint4 buf_load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// global [64 rows x Dh] tiles (row stride ss) -> registers; NCH 16-byte chunks per thread
template <int NCH> struct TileSrc {
  __amdgpu_buffer_rsrc_t rsrc;
  uint32_t off[NCH];     // this thread's chunks inside tile 0
  uint32_t tile_bytes;   // 64 rows
};
template <int DHP, int NT, int NCH>
__device__ __forceinline__ TileSrc<NCH> make_tilesrc(const bf16* g, int64_t ss, int S, int Dh, int tid) {
  constexpr int CPR = DHP / 8;
  TileSrc<NCH> t;
  t.rsrc = rows_rsrc(g, ss, S, Dh);
  t.tile_bytes = (uint32_t)(64 * ss * 2);
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int c = tid + i * NT;
    const int row = c / CPR, dc = c % CPR;
    t.off[i] = (c < 64 * CPR && dc * 8 < Dh) ? (uint32_t)((row * ss + dc * 8) * 2) : OOB_OFF;
  }
  return t;
}
template <int NCH>
__device__ __forceinline__ void stage_load(uint4 (&r)[NCH], const TileSrc<NCH>& t, int tile) {
  const uint32_t base = (uint32_t)tile * t.tile_bytes;
#pragma unroll
  for (int i = 0; i < NCH; i++) r[i] = buf_load16(t.rsrc, t.off[i] + base);
}
// chunk swizzle of a staged tile that is read both ways (see Strides): 16-byte chunk c of row r sits at chunk position
// c ^ swz_of<1>(r); swz_of<0> leaves the chunks in place
template <int SWZ>
__device__ __forceinline__ int swz_of(int row) {
  return SWZ == 1 ? (row >> 2) & 3 : 0;
}

template <int DHP, int NT, int NCH, int STRIDE, int SWZ>
__device__ __forceinline__ void stage_store(const uint4 (&r)[NCH], char* s, int tid) {
  constexpr int CPR = DHP / 8;
#pragma unroll
  for (int i = 0; i < NCH; i++) {
    const int c = tid + i * NT;
    const int row = c / CPR, dc = c % CPR;
    const int pc = dc ^ swz_of<SWZ>(row);
    if (c < 64 * CPR) *(uint4*)(s + row * STRIDE + pc * 16) = r[i];
  }
}

// Both fragment readers form their address as  tile + (a term of the lane alone) + (a compile-time constant): with r0 a
// multiple of 32 the swizzle of a row depends on the lane only and touches the two low bits of the chunk index, so one
// tile needs two lane terms per reader (k-step parity / row half) and everything else sits in the instruction's offset
// field.  Spelled out this way the loops hold a handful of address registers instead of one per fragment.
// row-wise operand fragment: element j = tile[r0 + (lane&31)][ks*16 + 8*(lane>>5) + j]   (r0 a multiple of 32)
template <int STRIDE, int SWZ>
__device__ __forceinline__ bf16x8 frag_rows(const char* s, int r0, int ks, int lane) {
  const int rl = lane & 31, hi = lane >> 5;
  const int w = swz_of<SWZ>(rl);
  const int low = (((ks * 2) & 3) | hi) ^ w;          // chunk index, low two bits: one lane term per parity of ks
  const int lane_off = rl * STRIDE + low * 16;
  const int imm = r0 * STRIDE + ((ks * 2) & ~3) * 16;
  return *(const bf16x8*)(s + lane_off + imm);
}
// column-wise operand fragment for a product whose other operand is an accumulator tile converted in
// place: element j = tile[r0 + 16*s2 + 8*(j>>2) + 4*(lane>>5) + (j&3)][c0 + (lane&31)]   (r0, c0 multiples of 32)
template <int STRIDE, int SWZ>
__device__ __forceinline__ bf16x8 frag_cols(const char* s, int r0, int s2, int c0, int lane) {
  const int hi = lane >> 5, l3 = lane & 3;
  const int rowl = 4 * hi + ((lane & 15) >> 2);       // the lane's row inside a 16-row group; its partner row is 8 below
  const int cl = 2 * ((lane >> 4) & 1) + (l3 >> 1);   // the lane's chunk inside a 32-column group
  const int sub = (l3 & 1) * 8;
  const int w_lo = SWZ == 1 ? hi : 0, w_hi = SWZ == 1 ? (hi | 2) : 0;   // swz_of(row), swz_of(row + 8)
  const int lane_lo = rowl * STRIDE + (cl ^ w_lo) * 16 + sub;
  const int lane_hi = (rowl + 8) * STRIDE + (cl ^ w_hi) * 16 + sub;
  const int imm = (r0 + 16 * s2) * STRIDE + (c0 >> 3) * 16;
  bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(s + lane_lo + imm));
  bf16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(s + lane_hi + imm));
  bf16x8 f;
  f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
  f[4] = hi4[0]; f[5] = hi4[1]; f[6] = hi4[2]; f[7] = hi4[3];
  return f;
}
// accumulator registers 8*s2 .. 8*s2+7 as the B operand of the next product (k-step s2)
__device__ __forceinline__ bf16x8 acc_to_frag(const f32x16& a, int s2) {
  bf16x8 f;
#pragma unroll
  for (int j = 0; j < 8; j++) f[j] = (bf16)a[8 * s2 + j];
  return f;
}
// stationary-side fragments straight from global: element j = g[row][ks*16 + 8*(lane>>5) + j]
template <int DHP>
__device__ __forceinline__ void load_stationary(bf16x8 (&f)[DHP / 16], const bf16* __restrict__ g, int64_t ss, int row,
                                                int S, int Dh, int lane) {
  const __amdgpu_buffer_rsrc_t rs = rows_rsrc(g, ss, S, Dh);
#pragma unroll
  for (int ks = 0; ks < DHP / 16; ks++) {
    const int d = ks * 16 + 8 * (lane >> 5);
    f[ks] = __builtin_bit_cast(bf16x8, buf_load16(rs, (row < S && d < Dh) ? (uint32_t)((row * ss + d) * 2) : OOB_OFF));
  }
}
// row index of accumulator register r inside a 32x32 tile (plus 4 for the upper 32 lanes)
__device__ __forceinline__ constexpr int acc_row(int r) { return (r & 3) + 8 * (r >> 2); }

// lanes l and l+32 exchange: returns {lower halves of a and b side by side, upper halves side by side}
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ float max_xor32(float x) {
  uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
  swap32(a, b);
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) bf16 bf16x2_t;
  bf16x2_t t;
  t[0] = (bf16)lo;
  t[1] = (bf16)hi;
  return __builtin_bit_cast(uint32_t, t);
}

// store a transposed accumulator set X^T[d][row] (row on the lane) as row-major bf16 rows, optional scale.  A lane holds
// 4 consecutive d per register quad and its partner lane (+-32) the next 4; quads of neighbouring groups are traded so
// that every lane writes 8 consecutive d with one 16-byte store.
template <int DHP>
__device__ __forceinline__ void store_rows(bf16* __restrict__ dst, const f32x16 (&acc)[DHP / 32], float mul, int Dh, int lane) {
#pragma unroll
  for (int dt = 0; dt < DHP / 32; dt++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t a01 = pack_bf16(acc[dt][8 * h + 0] * mul, acc[dt][8 * h + 1] * mul);
      uint32_t a23 = pack_bf16(acc[dt][8 * h + 2] * mul, acc[dt][8 * h + 3] * mul);
      uint32_t b01 = pack_bf16(acc[dt][8 * h + 4] * mul, acc[dt][8 * h + 5] * mul);
      uint32_t b23 = pack_bf16(acc[dt][8 * h + 6] * mul, acc[dt][8 * h + 7] * mul);
      swap32(a01, b01);
      swap32(a23, b23);
      const int d = dt * 32 + 16 * h + 8 * (lane >> 5);
      if (d < Dh) *(uint4*)(dst + d) = make_uint4(a01, a23, b01, b23);
    }
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // one v_exp_f32

#define ZERO16 {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}
#define MFMA __builtin_amdgcn_mfma_f32_32x32x16_bf16

// Workgroup -> (batch, head, block of stationary rows) for the streaming kernels, from a 1-D grid.  Workgroups are dealt
// to the 8 XCDs round-robin in launch order and every XCD has its own L2, so the blocks that share one head's streamed
// operands are given launch ids 8 apart: they run on the same XCD at about the same time, and the operands come from
// memory once per head instead of once per block.
struct HeadBlock {
  int64_t b, h;
  int xb;
  bool valid;
};
__device__ __forceinline__ HeadBlock head_block(int64_t B, int64_t H, int64_t nrows, int rows_per_block) {
  const int nxb = (int)((nrows + rows_per_block - 1) / rows_per_block);
  const int64_t per = 8 * (int64_t)nxb, L = blockIdx.x;
  const int64_t g = L / per, r = L - g * per;
  const int64_t hh = g * 8 + (r & 7);
  HeadBlock o;
  o.xb = (int)(r >> 3);
  o.valid = hh < B * H;
  o.b = hh / H;
  o.h = hh - o.b * H;
  return o;
}
static unsigned head_block_grid(int64_t B, int64_t H, int64_t S, int rows_per_block) {
  return (unsigned)(ceil_div(B * H, 8) * 8 * ceil_div(S, rows_per_block));
}
