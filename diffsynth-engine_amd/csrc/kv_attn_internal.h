// Shared by the two forms of the paged cache's attention (kv_attn.hip: few query rows; kv_attn_tile.hip: many).
#pragma once
#include "kv_internal.h"

namespace dsx {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  dsx_kv_cache c;
  dsx_kv_batch n;
  dsx_kv_attn_params p;
  int group;       // query heads per cache head
  int page_shift;
  int block_rows;  // packed query rows of a unit
  int nqb;         // query blocks per (sequence, cache head)
  int share;       // streaming form: 0, or the number of workgroups that share all units' tiles evenly
  int64_t first_split;  // tile form: units from this one on are cut
  int splits;           // into so many pieces of their key ranges
  float* part_o;   // (pieces, block_rows, 128) fp32
  float* part_ml;  // (pieces, block_rows, 2)
  Divisor by_group, by_nqb, by_batch, by_splits;
};

// Unit number -> (sequence, cache head, query block).  Sequences inside heads: runs of units (the tile form gives each XCD
// one) then hold all sequences alike, long and short.  Causal blocks come last first: they are the longest.
__device__ __forceinline__ void kv_unit(const AttnArgs& a, uint32_t unit, int& b, int& h, int& qb) {
  const uint32_t blocks = a.by_nqb(unit);
  qb = (int)(unit - blocks * a.nqb);
  if (a.p.causal) qb = a.nqb - 1 - qb;
  h = (int)a.by_batch(blocks);
  b = (int)(blocks - (uint32_t)h * a.n.batch);
}

// Inclusive sum over the lanes of a wave: six adds, each fed by the row shifts and broadcasts of the vector unit.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8: inside rows of 16
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast15 into rows 1 and 3
  v = dpp_add<0x143, 0xc>(v);  // row_bcast31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ float quad_max(float v) {  // over the four lanes n, n + 16, n + 32, n + 48
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const f16x2 v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// The factor that brings a partial sum with reference `m` to the reference `to` >= m.  A part that saw no token has
// reference -inf and sums of 0 (or NaN, which must survive): 0 unless nothing else saw one either.
__device__ __forceinline__ float join_factor(float m, float to) {
  return m == -INFINITY ? (to == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - to);
}

struct QFrag {
  i32x8 hi, lo;
  int s_hi, s_lo;
};

// Packed query row `pr` of a cache head: its span and its operand (the lane's elements 16g .. +15 and 64 + 16g .. +15).
struct QRaw {
  u32x4 w[4];
};
__device__ __forceinline__ void load_q(const AttnArgs& a, const KvSeq& s, int h, int pr, int g4, QRaw& raw, int& lo,
                                       int& hi) {
  const int row = a.by_group(pr), hh = h * a.group + pr - row * a.group;
  kv_row_span(s.kv, s.rows, row, a.p.causal, a.p.window, lo, hi);
  const uint16_t* src = (const uint16_t*)a.p.q + times(s.row0 + row, a.p.q_sr) + times(hh, a.p.q_sh) + 16 * g4;
#pragma unroll
  for (int w = 0; w < 4; ++w) raw.w[w] = *reinterpret_cast<const u32x4*>(src + 64 * (w >> 1) + 8 * (w & 1));
}
// q row -> two e4m3 terms and their e8m0 scales; the four lanes of a row share the exponent.  The converter divides by a
// power of two before it rounds, and multiplies on the way back.
__device__ __forceinline__ void split_q(const QRaw& raw, QFrag& f) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, raw.w[w][j] & 0x7fff7fffu));
  const uint32_t most = max((uint32_t)top[0], (uint32_t)top[1]);
  const float amax = quad_max(__uint_as_float(min(most, 0x7f80u) << 16));  // infinity if any element is not finite
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -110);
  const bool bad = !(amax < INFINITY);  // a scale of NaN: whatever the codes are, the scores are NaN
  if (bad) e = 0;
  const float up_hi = __uint_as_float((uint32_t)(127 + e) << 23), up_lo = __uint_as_float((uint32_t)(123 + e) << 23);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint32_t r0 = raw.w[w >> 1][2 * (w & 1)], r1 = raw.w[w >> 1][2 * (w & 1) + 1];
    const float x[4] = {bf16_lo(r0), bf16_hi(r0), bf16_lo(r1), bf16_hi(r1)};
    s16x2 hi = {0, 0}, lo = {0, 0};
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[0], x[1], up_hi, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[2], x[3], up_hi, true);
    f.hi[w] = __builtin_bit_cast(int, hi);
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(f.hi[w], up_hi, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(f.hi[w], up_hi, true);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0] - a[0], x[1] - a[1], up_lo, false);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2] - b[0], x[3] - b[1], up_lo, true);
    f.lo[w] = __builtin_bit_cast(int, lo);
  }
  f.s_hi = bad ? 255 : 127 + e;
  f.s_lo = bad ? 255 : 123 + e;
}

// A kernel's own argument block, read again where it is needed: what only the rare paths use would otherwise sit in
// scalar registers across the whole loop, and be spilled there.  (AttnArgs is the first argument of both kernels.)
__device__ __forceinline__ const AttnArgs& args_again() {
  auto p = (const __attribute__((address_space(4))) AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttnArgs*)p;
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {  // 0x80 in every byte that holds e4m3's NaN
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// The form for many query rows (kv_attn_tile.hip): 256 packed query rows per workgroup.
constexpr int kTileRows = 256;
int launch_kv_tile(const AttnArgs& a, int64_t units, hipStream_t st);
// Units at the end of the launch order whose key ranges are cut, and into how many pieces.
void kv_tile_split(int64_t units, int64_t span, int cus, int64_t& tail, int& pieces);

}  // namespace dsx
