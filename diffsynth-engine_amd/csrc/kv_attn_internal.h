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
};

// Unit number -> (sequence, cache head, query block).  Sequences inside heads: runs of units (the tile form gives each XCD
// one) then hold all sequences alike, long and short.  Causal blocks come last first: they are the longest.
__device__ __forceinline__ void kv_unit(const AttnArgs& a, uint32_t unit, int& b, int& h, int& qb) {
  qb = (int)(unit % (uint32_t)a.nqb);
  if (a.p.causal) qb = a.nqb - 1 - qb;
  unit /= (uint32_t)a.nqb;
  b = (int)(unit % (uint32_t)a.n.batch);
  h = (int)(unit / (uint32_t)a.n.batch);
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

// q row -> two e4m3 terms and their e8m0 scales.  x: the lane's 32 elements; the four lanes of a row share the exponent.
struct QFrag {
  i32x8 hi, lo;
  int s_hi, s_lo;
};
__device__ __forceinline__ void split_q(const float (&x)[32], QFrag& f) {
  float amax = 0.f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    amax = fmaxf(amax, fabsf(x[j]));
    odd |= !(fabsf(x[j]) < INFINITY);
  }
  amax = quad_max(odd ? INFINITY : amax);
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -110);
  const bool bad = !(amax < INFINITY);
  if (bad) e = 0;
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e, a normal number for e in [-110, 120]
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = bad ? 0.f : x[4 * w + j] * down;
    const uint32_t hi = pack_e4m3x4_inrange(y[0], y[1], y[2], y[3]);
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, true);
    f.hi[w] = (int)hi;
    f.lo[w] = (int)pack_e4m3x4_inrange(16.f * (y[0] - a[0]), 16.f * (y[1] - a[1]), 16.f * (y[2] - b[0]),
                                       16.f * (y[3] - b[1]));
  }
  f.s_hi = bad ? 255 : 127 + e;
  f.s_lo = bad ? 255 : 127 + e - 4;
}

// Packed query row `pr` of a cache head: its span and its operand (the lane's elements 16g .. +15 and 64 + 16g .. +15).
struct QRaw {
  u32x4 w[4];
};
__device__ __forceinline__ void load_q(const AttnArgs& a, const KvSeq& s, int h, int pr, int g4, QRaw& raw, int& lo,
                                       int& hi) {
  const int row = pr / a.group, hh = h * a.group + pr % a.group;
  kv_row_span(s.kv, s.rows, row, a.p.causal, a.p.window, lo, hi);
  const uint16_t* src = (const uint16_t*)a.p.q + (int64_t)(s.row0 + row) * a.p.q_sr + hh * a.p.q_sh + 16 * g4;
#pragma unroll
  for (int w = 0; w < 4; ++w) raw.w[w] = *reinterpret_cast<const u32x4*>(src + 64 * (w >> 1) + 8 * (w & 1));
}
__device__ __forceinline__ void split_q(const QRaw& raw, QFrag& f) {
  float x[32];
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[8 * w + 2 * j] = bf16_lo(raw.w[w][j]);
      x[8 * w + 2 * j + 1] = bf16_hi(raw.w[w][j]);
    }
  split_q(x, f);
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
