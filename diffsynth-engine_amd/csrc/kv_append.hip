// Appending a batch's keys and values to the paged 8-bit cache, and its queries' normalisation and rotation.
//
// One workgroup = one (page, head) block of K or of V, or 16 rows x kQHeads heads of q.  A block's tokens are held in
// registers between the two passes over them (largest magnitude, then codes), so each element is read once and written
// once: 16 lanes per token, 8 elements per lane, page/16 tokens per lane.  A row of q keeps its line of the rotation table in
// registers for kQHeads heads (one head a row: 73 instead of 57 us at 8 x 2001 tokens).
// Bound: HBM, 2 bytes in and 1 out an element of k and v, 2 and 2 of q.  8 x 2001 tokens, 8 heads, 32 of q: 57 us, 260 MB
// (4.5 TB/s where a large copy reaches 4.9); 4680 tokens, 40 heads, without q: 30 us, 144 MB (4.7 TB/s); single tokens: the
// launch, lengths, rows and the store in a row, 4.3 us.
#include <stdlib.h>

#include <algorithm>

#include "kv_internal.h"

namespace dsx {
namespace {

constexpr int kQHeads = 4;

struct AppendArgs {
  dsx_kv_cache c;
  dsx_kv_batch n;
  dsx_kv_append_params p;
  int page_shift;
  int blocks_per_seq;  // pages that max_rows rows can reach
  int64_t q_begin;     // first workgroup of the q part
  int q_per_seq, q_per_row;  // workgroups a sequence, kQHeads heads a row
  Divisor by_heads, by_blocks, by_q_per_seq, by_q_per_row;
};

__device__ __forceinline__ float row16_sum(float v) {  // over the 16 lanes of a token
  v += dpp_f32<kDppRowRor8>(v);
  v += dpp_f32<kDppRowRor4>(v);
  v += dpp_f32<kDppQuadXor2>(v);
  v += dpp_f32<kDppQuadXor1>(v);
  return v;
}

__device__ __forceinline__ void load8(const uint16_t* src, float (&x)[8]) {
  const u32x4 w = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = bf16_lo(w[j]);
    x[2 * j + 1] = bf16_hi(w[j]);
  }
}

// RMSNorm over the head, then the rotation of pairs (2i, 2i + 1): the lane's place in the token's 16 is its elements 8 ln ..
// and cs the (cos, sin) of its four pairs.
__device__ __forceinline__ void load_turn(const float* rope_row, int ln, float (&cs)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(rope_row + 8 * ln);
  const f32x4 b = *reinterpret_cast<const f32x4*>(rope_row + 8 * ln + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cs[j] = a[j];
    cs[4 + j] = b[j];
  }
}
__device__ __forceinline__ void turn(float (&x)[8], const float (&cs)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x0 = x[2 * j], x1 = x[2 * j + 1], c = cs[2 * j], s = cs[2 * j + 1];
    x[2 * j] = x0 * c - x1 * s;
    x[2 * j + 1] = x0 * s + x1 * c;
  }
}
__device__ __forceinline__ void norm(float (&x)[8], const float (&g)[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
  const float r = __builtin_amdgcn_rsqf(row16_sum(ss) * (1.0f / kKvDim) + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] *= r * g[j];
}

// value * 2^-e as the clamp's operand: saturates at +-448 (infinities too), NaN stays NaN
__device__ __forceinline__ float clamp448(float v) {
  const float y = fminf(fmaxf(v, -448.f), 448.f);
  return v == v ? y : v;
}

template <int TOK>  // tokens per 16-lane group = page / 16
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const dsx_kv_cache& c = a.c;
  const dsx_kv_batch& n = a.n;
  const dsx_kv_append_params& p = a.p;
  const int tid = threadIdx.x, ln = tid & 15, grp = tid >> 4;
  __shared__ uint32_t smax[4];
  asm volatile("" ::"s"(c.k), "s"(n.row_start), "s"(p.k), "s"(p.q_norm_w), "s"(p.total_rows), "s"(a.q_begin));

  if ((int64_t)blockIdx.x >= a.q_begin) {
    const unsigned u = blockIdx.x - (unsigned)a.q_begin;
    const int b = a.by_q_per_seq(u), chunk = (int)u - b * a.q_per_seq;
    const KvSeq s = kv_seq(n, b, p.total_rows);
    if (!s.ok || s.kv < s.rows) return;
    const int at = chunk * 16 + grp, row = a.by_q_per_row(at), h0 = (at - row * a.q_per_row) * kQHeads;
    if (row >= s.rows) return;
    const uint16_t* src = (const uint16_t*)p.q + times(s.row0 + row, p.q_sr) + 8 * ln;
    uint16_t* dst = (uint16_t*)p.q_out + times(s.row0 + row, p.qo_sr) + 8 * ln;
    float x[kQHeads][8], g[8], cs[8];
#pragma unroll
    for (int i = 0; i < kQHeads; ++i) load8(src + times(min(h0 + i, p.heads_q - 1), p.q_sh), x[i]);
    if (p.q_norm_w) load8((const uint16_t*)p.q_norm_w + 8 * ln, g);
    if (p.rope) load_turn(p.rope + b * p.rope_sb + (int64_t)(s.kv - s.rows + row) * kKvDim, ln, cs);
#pragma unroll
    for (int i = 0; i < kQHeads; ++i) {
      if (p.q_norm_w) norm(x[i], g, p.norm_eps);
      if (p.rope) turn(x[i], cs);
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(x[i][2 * j], x[i][2 * j + 1]);
      if (h0 + i < p.heads_q) *reinterpret_cast<u32x4*>(dst + times(h0 + i, p.qo_sh)) = w;
    }
    return;
  }

  // ---- one (page, head) block of K or V
  const unsigned u = a.by_heads(blockIdx.x);
  const int h = (int)(blockIdx.x - u * c.heads);
  const bool is_v = u & 1;
  const int b = a.by_blocks(u >> 1), j = (int)(u >> 1) - b * a.blocks_per_seq;
  const KvSeq s = kv_seq(n, b, p.total_rows);
  if (!s.ok || s.kv < s.rows) return;
  const int first = s.kv - s.rows;  // the first appended token
  const int page = c.page_size;
  const int pi = (first >> a.page_shift) + j;
  const int base = pi << a.page_shift;  // the block's first token
  if (base >= s.kv || s.rows == 0) return;
  const int id = n.page_table[times(b, n.table_sb) + pi];
  const int lo = first > base ? first - base : 0;  // tokens [lo, hi) of the block are new, [0, lo) stay
  const int hi = s.kv - base < page ? s.kv - base : page;

  const uint16_t* src = is_v ? (const uint16_t*)p.v + times(h, p.v_sh) : (const uint16_t*)p.k + times(h, p.k_sh);
  const int64_t sr = is_v ? p.v_sr : p.k_sr;
  float x[TOK][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < TOK; ++i) {
    const int t = grp + 16 * i;
    if (t >= lo && t < hi) {
      load8(src + times(s.row0 + base + t - first, sr) + 8 * ln, x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
    }
  }
  // (the rows are under way before the page number that they go to is looked at)
  if (id < 0 || id >= c.pages) return;
  uint8_t* codes = is_v ? (uint8_t*)c.v + times(id, c.v_sp) + h * c.v_sh : (uint8_t*)c.k + times(id, c.k_sp) + h * c.k_sh;
  uint8_t* scale = is_v ? (uint8_t*)c.v_scale + times(id, c.vs_sp) + h : (uint8_t*)c.k_scale + times(id, c.ks_sp) + h;
  if (!is_v && p.k_norm_w) {
    float g[8];
    load8((const uint16_t*)p.k_norm_w + 8 * ln, g);
#pragma unroll
    for (int i = 0; i < TOK; ++i) norm(x[i], g, p.norm_eps);
  }
  if (!is_v && p.rope) {
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const int t = grp + 16 * i;
      if (t >= lo && t < hi) {
        float cs[8];
        load_turn(p.rope + b * p.rope_sb + (int64_t)(base + t) * kKvDim, ln, cs);
        turn(x[i], cs);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TOK; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = fabsf(x[i][e]);
      amax = fmaxf(amax, v < INFINITY ? v : 0.f);
    }
  amax = wave_max(amax);
  if ((tid & 63) == 0) smax[tid >> 6] = __float_as_uint(amax);  // (non-negative floats order as their bits)
  __syncthreads();
  const uint32_t top = max(max(smax[0], smax[1]), max(smax[2], smax[3]));
  int e = kv_block_exponent(top);
  if (lo > 0) {
    const int old = (int)*scale - 127;
    if (old > e) {
      e = old;
    } else if (old < e) {  // the kept codes move to the larger scale: exact but for what becomes subnormal
#pragma unroll
      for (int i = 0; i < TOK; ++i) {
        const int t = grp + 16 * i;
        if (t < lo) {
          u32x2* at = reinterpret_cast<u32x2*>(codes + t * kKvDim + 8 * ln);
          u32x2 w = *at;
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            float f[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) f[q] = ldexpf(e4m3_bits_to_f32((w[d] >> (8 * q)) & 0xffu), old - e);
            w[d] = pack_e4m3x4_inrange(f[0], f[1], f[2], f[3]);
          }
          *at = w;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TOK; ++i) {
    const int t = grp + 16 * i;
    if (t >= lo && t < hi) {
      u32x2 w;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        float f[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) f[q] = clamp448(ldexpf(x[i][4 * d + q], -e));
        w[d] = pack_e4m3x4_inrange(f[0], f[1], f[2], f[3]);
      }
      *reinterpret_cast<u32x2*>(codes + t * kKvDim + 8 * ln) = w;
    }
  }
  __syncthreads();  // every lane has read the old exponent
  if (tid == 0) *scale = (uint8_t)(e + 127);
}

bool below_2_31(int64_t x) { return x >= 0 && x <= 0x7fffffff; }

}  // namespace

bool kv_rows_ok(const void* p, int64_t sr, int64_t sh) {
  return ((uintptr_t)p & 15) == 0 && sr % 8 == 0 && sh % 8 == 0 && below_2_31(sr) && below_2_31(sh);
}

int kv_check_cache(const dsx_kv_cache* c, const dsx_kv_batch* n, int64_t total_rows) {
  if (!c || !n) return DSX_ENULL;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || !n->page_table || !n->row_start || !n->kv_len) return DSX_ENULL;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return DSX_EBADSHAPE;
  if (c->pages < 1 || c->heads < 1 || n->batch < 1 || n->table_pages < 1 || n->table_sb < n->table_pages ||
      n->max_rows < 0 || n->max_rows > (1 << 30) || n->max_kv_len < 0 || n->max_kv_len > (1 << 30) || total_rows < 0 ||
      total_rows > 0x7fffffff || n->max_kv_len > (int64_t)n->table_pages * c->page_size)
    return DSX_EBADSHAPE;
  if (!below_2_31(c->k_sp) || !below_2_31(c->v_sp) || !below_2_31(c->ks_sp) || !below_2_31(c->vs_sp) ||
      !below_2_31(n->table_sb))
    return DSX_EBADSHAPE;
  if (c->k_sp % 16 || c->k_sh % 16 || c->v_sp % 16 || c->v_sh % 16) return DSX_EALIGN;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return DSX_EALIGN;
  if (((uintptr_t)n->page_table | (uintptr_t)n->row_start | (uintptr_t)n->kv_len) & 3) return DSX_EALIGN;
  return DSX_OK;
}

}  // namespace dsx

extern "C" int dsx_kv_append(const dsx_kv_cache* cache, const dsx_kv_batch* batch, const dsx_kv_append_params* p,
                             void* stream) {
  using namespace dsx;
  if (!p) return DSX_ENULL;
  const int rc = kv_check_cache(cache, batch, p->total_rows);
  if (rc != DSX_OK) return rc;
  const dsx_kv_cache& c = *cache;
  const dsx_kv_batch& n = *batch;
  if (!p->k || !p->v || (p->q && !p->q_out)) return DSX_ENULL;
  if (p->q && p->heads_q < 1) return DSX_EBADSHAPE;
  if (!(p->norm_eps >= 0.f)) return DSX_EBADSHAPE;
  if (!kv_rows_ok(p->k, p->k_sr, p->k_sh) || !kv_rows_ok(p->v, p->v_sr, p->v_sh)) return DSX_EALIGN;
  if (p->q && (!kv_rows_ok(p->q, p->q_sr, p->q_sh) || !kv_rows_ok(p->q_out, p->qo_sr, p->qo_sh))) return DSX_EALIGN;
  if (((uintptr_t)p->k_norm_w | (uintptr_t)p->q_norm_w | (uintptr_t)p->rope) & 15) return DSX_EALIGN;
  if (p->rope && (p->rope_rows < n.max_kv_len || p->rope_sb % 4 ||
                  (p->rope_sb != 0 && p->rope_sb < p->rope_rows * kKvDim)))
    return DSX_EBADSHAPE;
  if (n.max_rows == 0 || p->total_rows == 0) return DSX_OK;
  AppendArgs a{};
  a.c = c;
  a.n = n;
  a.p = *p;
  a.page_shift = __builtin_ctz((unsigned)c.page_size);
  const int64_t rows = std::min<int64_t>({n.max_rows, n.max_kv_len, p->total_rows});
  if (rows == 0) return DSX_OK;
  a.blocks_per_seq = (int)((rows + c.page_size - 2) / c.page_size + 1);
  const int64_t kv_wgs = (int64_t)n.batch * a.blocks_per_seq * c.heads * 2;
  a.q_begin = kv_wgs;
  const int64_t q_per_seq = p->q ? (rows * ((p->heads_q + kQHeads - 1) / kQHeads) + 15) / 16 : 0;
  const int64_t total = kv_wgs + (int64_t)n.batch * q_per_seq;
  if (total >= (1ll << 24)) return DSX_EBADSHAPE;  // a launch has fewer than 2^32 threads
  a.q_per_seq = (int)q_per_seq;
  a.q_per_row = (p->heads_q + kQHeads - 1) / kQHeads;
  a.by_heads = Divisor::of(c.heads);
  a.by_blocks = Divisor::of(a.blocks_per_seq);
  if (q_per_seq > 0) {
    a.by_q_per_seq = Divisor::of(a.q_per_seq);
    a.by_q_per_row = Divisor::of(a.q_per_row);
  }
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)total), block(256);
  switch (c.page_size) {
    case 16: kv_append_kernel<1><<<grid, block, 0, st>>>(a); break;
    case 32: kv_append_kernel<2><<<grid, block, 0, st>>>(a); break;
    case 64: kv_append_kernel<4><<<grid, block, 0, st>>>(a); break;
    default: kv_append_kernel<8><<<grid, block, 0, st>>>(a); break;
  }
  return hipGetLastError() == hipSuccess ? DSX_OK : DSX_ELAUNCH;
}

extern "C" int dsx_kv_plan_check(const dsx_kv_batch* n, int32_t pages, int32_t page_size, int64_t total_rows,
                                 int for_append, int32_t* bad_sequence) {
  using namespace dsx;
  if (!n || !n->page_table || !n->row_start || !n->kv_len) return DSX_ENULL;
  if (page_size < 1 || pages < 1 || n->batch < 1 || n->table_pages < 1 || n->table_sb < n->table_pages)
    return DSX_EBADSHAPE;
  int32_t none;
  int32_t& bad = bad_sequence ? *bad_sequence : none;
  for (int b = 0; b < n->batch; ++b) {
    bad = b;
    const KvSeq s = kv_seq(*n, b, total_rows);
    if (!s.ok || s.kv > (int64_t)n->table_pages * page_size) return DSX_EBADSHAPE;
    if (for_append && s.kv < s.rows) return DSX_EBADSHAPE;
    const int32_t* row = n->page_table + b * n->table_sb;
    for (int t = 0; t < ((int64_t)s.kv + page_size - 1) / page_size; ++t)
      if (row[t] < 0 || row[t] >= pages) return DSX_EBADSHAPE;
  }
  if (for_append) {  // a page that is written belongs to one place of one sequence
    uint8_t* listed = (uint8_t*)calloc((size_t)pages, 1);
    if (!listed) return DSX_EWORKSPACE;
    int rc = DSX_OK;
    for (int pass = 0; pass < 2 && rc == DSX_OK; ++pass)
      for (int b = 0; b < n->batch && rc == DSX_OK; ++b) {
        const KvSeq s = kv_seq(*n, b, total_rows);
        const int32_t* row = n->page_table + b * n->table_sb;
        const int end = (int)(((int64_t)s.kv + page_size - 1) / page_size);
        const int begin = pass == 0 ? 0 : s.rows == 0 ? end : (s.kv - s.rows) / page_size;
        for (int t = begin; t < end; ++t) {
          uint8_t& times = listed[row[t]];
          if (pass == 0) {
            times = times < 2 ? times + 1 : 2;
          } else if (times > 1) {
            bad = b;
            rc = DSX_EBADSHAPE;
          }
        }
      }
    free(listed);
    if (rc != DSX_OK) return rc;
  }
  bad = -1;
  return DSX_OK;
}
