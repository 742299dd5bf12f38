// Attention over the paged 8-bit key/value cache.
//
// Work: a unit is (sequence, cache head, block of query rows), where the query rows of a cache head are its
// heads_q / heads query heads times the sequence's rows, packed as row * group + head.  A workgroup walks a piece of the
// unit's key range in tiles of 32 keys, one wave per tile, each of its eight waves with a running maximum, sum and
// output of its own; they meet in LDS at the end, the pieces of a split key range in a second kernel.
//
// S^T = K Q^T on v_mfma_scale_f32_16x16x128_f8f6f4: K's codes are the operand as they lie in the cache, the page's
// e8m0 scale rides in the instruction's scale operand, and q is the sum of two e4m3 terms with scales of their own (hi:
// rounded at the row's block exponent; lo: the remainder times 16, which has at most four significant bits, so the sum is
// exact down to 2^-22 of the row's largest element).  Two fp8 products of 128 elements take the matrix pipe as long as
// the four bf16 products that expanding K would need, and K is never expanded.
// O^T += V^T P^T on v_mfma_f32_16x16x32_f16: V's codes are exact in fp16, and the weights get fp16's eleven bits
// instead of bf16's eight.  fp16's range is kept safe by the weight's unit: with e_v the exponent of the block's scale,
//   w = exp2(s c + e_v + 14 - m),  m = running maximum of s c + e_v   (c = softmax_scale log2 e),
// lies in (0, 2^14] and multiplies the raw codes; the row sum adds 2^-e_v w, before w is rounded.  |e_v| <= 48 bounds what
// two blocks can be apart to 2^96: in fp32 (row sums, factors that join partial sums) a weight leaves the normal range
// (2^-126) only for tokens whose share of the softmax is below 2^-30.  The fp16 weight is within 2^-11 of itself or 2^-25,
// half its smallest step: beside 2^-11 sum_j p_j |v_j| an output is off by at most
//   2^-39 max_j(p_j 2^e_j) sum_j |code_j|   over the tokens j that the row sees
// (tile form: 2^-33; with pages of 16 and 32, where a weight may be rounded twice: 2^-32, beside 2^-10 sum_j p_j |v_j|).
// So precision is relative to the largest p_j 2^e_j, and not to a token's share alone: beside a token of the same score in a
// block whose scale is 2^28 (2^22) as large a weight loses bits, at 2^40 (2^34) all of them.  Weights relative to the share
// would lose the reverse, tokens of a small share in blocks of a large scale, and those dominate the output.
// Lane (n = lane % 16, g = lane / 16) of S^T holds query n, keys 4g .. 4g + 3 of a 16-key half: packed to fp16, the two
// halves of a tile are the B operand of the second product as they stand.
// A masked tile may hold NaN codes of tokens that some rows do not see: 0 * NaN must not reach those rows, so such a
// tile takes V with the NaN replaced by 0 and adds NaN to the rows that do see it (a second product over indicators).
//
// Bound: HBM, 256 bytes a token and cache head for a handful of flops each; codes go from memory to registers in whole
// 128-byte lines and nothing is staged.  A read of the same pages without any arithmetic reaches 6.0 TB/s; 1 x 131071
// tokens, 40 heads: 228 us and 5 for the join (5.8 TB/s); 64 sequences to 16384 tokens, 8 heads: 276 + 5 us (5.8 TB/s).
// Eight waves of 228 to 256 registers fill a compute unit (with four of them the 131071 tokens took 282 us instead of 258).
// Short caches are bound by the chain launch -> lengths -> page numbers -> scales and codes -> products -> join of the
// waves: 1 x 1561 tokens, 12 heads: 7.1 us and 3.5 for the join of the pieces.  Hence first pages beside the lengths, codes
// beside the scales, q's split beside both, and no division anywhere (8.8 + 3.9 us before).
#include <algorithm>
#include <type_traits>

#include "kv_attn_internal.h"

namespace dsx {
namespace {

constexpr int kTileKeys = 32;
constexpr float kHeadroom = 14.f;  // log2 of the largest fp16 weight

// A tile's codes in flight.  K: row n of each 16-key half, elements 16g .. +15 and 64 + 16g .. +15.  V: tokens 4g + t,
// elements 8n .. 8n + 7.
struct TileRegs {
  u32x4 k[2][2];
  u32x2 v[2][4];
};

constexpr int kWaves = 8;

struct StreamLds {  // the waves' results
  float o[kWaves][16][kKvDim + 4];
  float m[kWaves][16], l[kWaves][16];
};

// ---- Equal shares.  The tiles of all units lie behind one another, head by head and sequence by sequence, and are dealt
// to `share` workgroups in equal runs whatever the sequences' lengths (which only the device knows): a run may end inside
// a unit, and then both sides leave partial results.  Every wave sums the lengths for itself, a sequence per lane.
__device__ __forceinline__ int span_tiles(const AttnArgs& a, const KvSeq& s) {  // tiles that any row of a sequence sees
  int lo, hi, unused;
  kv_row_span(s.kv, s.rows, 0, a.p.causal, a.p.window, lo, unused);
  kv_row_span(s.kv, s.rows, s.rows - 1, a.p.causal, a.p.window, unused, hi);
  return s.rows == 0 ? 0 : max((hi + kTileKeys - 1) / kTileKeys - lo / kTileKeys, 0);
}
struct Lens {     // 64 sequences from b0 on, one per lane
  int b0, count, upto;  // the lane's tiles; the sum over the lanes up to it
  KvSeq s;
};
__device__ __forceinline__ void load_lens(const AttnArgs& a, int b0, int lane, Lens& x) {
  x.b0 = b0;
  x.s = kv_seq(a.n, min(b0 + lane, a.n.batch - 1), a.p.total_rows);
  x.count = b0 + lane < a.n.batch ? span_tiles(a, x.s) : 0;
  x.upto = wave_scan(x.count);
}
__device__ __forceinline__ int head_sum(const AttnArgs& a, int lane, Lens& x) {  // tiles of one head; leaves x at b0 = 0
  int sum = 0;
  for (int b0 = (a.n.batch - 1) & ~63; b0 >= 0; b0 -= 64) {
    load_lens(a, b0, lane, x);
    sum += __builtin_amdgcn_readlane(x.upto, 63);
  }
  return sum;
}
// Runs of `total` tiles: workgroup w of n takes [share_begin(w), share_begin(w + 1)).  No run is shorter than two tiles a
// wave: below that, what a piece costs besides its tiles is most of its time.
__device__ __forceinline__ int share_count(int total, int n) { return min(n, max(total / (2 * kWaves), 1)); }
__device__ __forceinline__ int share_begin(int total, int n, int w) { return w * (total / n) + w * (total % n) / n; }
__device__ __forceinline__ int share_of(int total, int n, int x) {  // whose run holds tile x
  return (int)((((uint64_t)x + 1) * n - 1) / (uint64_t)total);
}

// NQ: 16-row columns of query rows.  BLOCKS: (page, head) blocks that a tile may lie in, 2 for pages of 16 tokens.
// SHARE: even shares (a.share), or a.splits pieces of every unit.
template <int NQ, int BLOCKS, bool SHARE>
__global__ __launch_bounds__(64 * kWaves, 2) void kv_stream_kernel(AttnArgs a) {
  const dsx_kv_cache& c = a.c;
  const int wave = uniform(threadIdx.x >> 6);
  // The lane's number, anew where it is asked for: sums of it for the end of the kernel would be made at its beginning and
  // held, or spilled, across the tiles.
  auto this_lane = [&]() __attribute__((always_inline)) {
    int x = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(x));
    return x;
  };
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  StreamLds* sm = reinterpret_cast<StreamLds*>(smem);
  // All of the argument block at once: five cache lines, which would be met one after another.
  asm volatile("" ::"s"(a.c.k), "s"(a.n.row_start), "s"(a.p.q), "s"(a.p.total_rows), "s"(a.part_o));

  // This workgroup's tiles among all of them, as head and place in the head (one whole unit: nothing to look up).
  int h = 0, place = 0, left = 1, head_tiles = 1;
  Lens lens;
  if constexpr (SHARE) {
    head_tiles = head_sum(a, this_lane(), lens);
    const int total = head_tiles * c.heads;
    if (total == 0) return;
    const int n = share_count(total, a.share);
    if ((int)blockIdx.x >= n) return;
    place = share_begin(total, n, blockIdx.x);
    left = share_begin(total, n, blockIdx.x + 1) - place;
    h = place / head_tiles;
    place -= h * head_tiles;
  }
  for (bool again = false; left > 0; again = true) {
  const int lane = this_lane(), n16 = lane & 15, g4 = lane >> 4;
  // ---- the next segment: a whole unit or a part of one
  int b, qb = 0, skip = 0, count = 0x3fffffff, piece = -1;  // piece: where a part's result goes
  int first = wave, stride = kWaves;  // the wave's tiles among the segment's
  KvSeq s;
  // Without a window the first pages are known before the lengths are, and asked for along with them.
  const bool early = !SHARE && a.p.window == 0;
  int pg[BLOCKS] = {};
  if constexpr (SHARE) {
    if (place == head_tiles) {
      place = 0;
      ++h;
    }
    int before = 0;  // tiles of the sequences in front of the 64 at hand
    uint64_t beyond;
    if (lens.b0 != 0) load_lens(a, 0, lane, lens);
    while ((beyond = __builtin_amdgcn_ballot_w64(before + lens.upto > place)) == 0) {
      if (lens.b0 + 64 >= a.n.batch) return;  // (lengths that another stream changed under the kernel)
      before += __builtin_amdgcn_readlane(lens.upto, 63);
      load_lens(a, lens.b0 + 64, lane, lens);
    }
    const int at = __builtin_ctzll(beyond);
    b = lens.b0 + at;
    s.row0 = __builtin_amdgcn_readlane(lens.s.row0, at);
    s.rows = __builtin_amdgcn_readlane(lens.s.rows, at);
    s.kv = __builtin_amdgcn_readlane(lens.s.kv, at);
    s.ok = true;  // (one that is not has no tiles)
    const int all = __builtin_amdgcn_readlane(lens.count, at);
    skip = place - (before + __builtin_amdgcn_readlane(lens.upto, at) - all);
    count = min(all - skip, left);
    if (count < all) piece = 2 * blockIdx.x + (skip == 0);
    place += count;
    left -= count;
  } else {
    const int unit = a.by_splits(blockIdx.x);
    kv_unit(a, unit, b, h, qb);
    b = uniform(b);
    if (a.splits > 1) {  // a piece takes every a.splits-th run of eight tiles: its first page needs no length
      first += kWaves * (int)(blockIdx.x - unit * a.splits);
      stride *= a.splits;
      piece = blockIdx.x;
    }
    if (early) {
#pragma unroll
      for (int hf = 0; hf < BLOCKS; ++hf)
        pg[hf] = a.n.page_table[times(b, a.n.table_sb) +
                                min(((first + stride * lane) * kTileKeys + 16 * hf) >> a.page_shift, a.n.table_pages - 1)];
    }
    s = kv_seq(a.n, b, a.p.total_rows);
    left = 0;
  }
  // (one value each for the whole wave, which divisions and loads leave in vector registers)
  b = uniform(b);
  h = uniform(h);
  qb = uniform(qb);
  s = {uniform(s.row0), uniform(s.rows), uniform(s.kv), uniform((int)s.ok) != 0};
  const int packed = s.rows * a.group;
  const int pr0 = qb * 16 * NQ;
  if (pr0 >= packed) return;
  if (again) __syncthreads();  // the LDS of the segment before

  // ---- the rows of this block and the keys any of them sees
  const int row_lo = a.by_group(pr0), row_hi = a.by_group(min(pr0 + 16 * NQ, packed) - 1);
  int lo_first, hi_first, lo_last, hi_last;
  kv_row_span(s.kv, s.rows, row_lo, a.p.causal, a.p.window, lo_first, hi_first);
  kv_row_span(s.kv, s.rows, row_hi, a.p.causal, a.p.window, lo_last, hi_last);
  const int tile_end = (hi_last + kTileKeys - 1) / kTileKeys;
  const int t_begin = lo_first / kTileKeys + skip;
  const int t_end = min(t_begin + count, tile_end);
  // This wave's tiles t_first + stride i, i in [0, tiles); all rows see all keys of those in [in_lo, in_hi).
  const int t_first = t_begin + first;
  auto tiles_below = [&](int t) -> int {
    const unsigned rounds = (unsigned)(t - t_first + stride - 1) / (unsigned)kWaves;
    return t <= t_first ? 0 : SHARE ? rounds : a.by_splits(rounds);
  };
  const int tiles = tiles_below(t_end);
  const int in_lo = min(tiles_below((lo_last + kTileKeys - 1) / kTileKeys), tiles);
  const int in_hi = max(min(tiles_below(hi_first / kTileKeys), tiles), in_lo);

  QRaw raw[NQ];
  int my_lo[NQ], my_hi[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    load_q(a, s, h, min(pr0 + q * 16 + n16, packed - 1), g4, raw[q], my_lo[q], my_hi[q]);

  const uint8_t* kbase = (const uint8_t*)c.k + (int64_t)h * c.k_sh;
  const uint8_t* vbase = (const uint8_t*)c.v + (int64_t)h * c.v_sh;
  const uint32_t koff = n16 * kKvDim + 16 * g4, voff = 4 * g4 * kKvDim + 8 * n16;
  const int page_mask = c.page_size - 1;

  // Page numbers and scales of 64 of the wave's tiles, one tile per lane: two dependent loads per 64 tiles instead of two
  // per tile.  scales: k of the blocks in bytes 0, 1, v in bytes 2, 3.  Keys behind the last one take its page: what is
  // loaded for them is not used.  (Asked for early, they take the entry that the table has, or its last.)
  int pg_at = -1;
  uint32_t sc_all = 0;
  uint32_t ks[BLOCKS], vs[BLOCKS];  // scale bytes on their way
  bool bad[BLOCKS];
  auto ask_pages = [&](int chunk, bool have) __attribute__((always_inline)) {
    const AttnArgs& r = args_again();
    pg_at = chunk;
    if (!have) {
#pragma unroll
      for (int hf = 0; hf < BLOCKS; ++hf) {
        const int key = min((t_first + stride * (64 * chunk + lane)) * kTileKeys + 16 * hf, hi_last - 1);
        pg[hf] = r.n.page_table[times(b, r.n.table_sb) + (key >> r.page_shift)];
      }
    }
#pragma unroll
    for (int hf = 0; hf < BLOCKS; ++hf) {
      bad[hf] = pg[hf] < 0 || pg[hf] >= r.c.pages;
      pg[hf] = bad[hf] ? 0 : pg[hf];
      ks[hf] = ((const uint8_t*)r.c.k_scale)[times(pg[hf], r.c.ks_sp) + h];
      vs[hf] = ((const uint8_t*)r.c.v_scale)[times(pg[hf], r.c.vs_sp) + h];
    }
  };
  auto take_scales = [&]() __attribute__((always_inline)) {
    sc_all = 0;
#pragma unroll
    for (int hf = 0; hf < BLOCKS; ++hf) {
      // (no scale: NaN scores for every row that sees the block, and nothing for the others)
      const bool none = bad[hf] || vs[hf] == 255;
      sc_all |= ((none ? 255u : ks[hf]) << (8 * hf)) | ((none ? 127u : vs[hf]) << (16 + 8 * hf));
    }
  };
  auto scales_at = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)sc_all, i & 63); };
  auto load_codes = [&](int i, TileRegs& r) __attribute__((always_inline)) {
    const int key = (t_first + stride * i) * kTileKeys;
    uint32_t ko = koff, vo = voff;
    asm volatile("" : "+v"(ko), "+v"(vo));  // (32-bit offsets to a scalar base; widened outside, they would be 64-bit sums)
    const uint8_t *kp, *vp;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      if (hf < BLOCKS) {
        const int page = __builtin_amdgcn_readlane(pg[hf], i & 63);
        const int tok = (key + 16 * hf) & page_mask;
        kp = kbase + times(page, c.k_sp) + tok * kKvDim;
        vp = vbase + times(page, c.v_sp) + tok * kKvDim;
      }
      const int more = hf < BLOCKS ? 0 : 16 * kKvDim;
#pragma unroll
      for (int w = 0; w < 2; ++w) r.k[hf][w] = *reinterpret_cast<const u32x4*>(kp + ko + 64 * w + more);
#pragma unroll
      for (int t = 0; t < 4; ++t) r.v[hf][t] = *reinterpret_cast<const u32x2*>(vp + vo + t * kKvDim + more);
    }
  };
  auto load_tile = [&](int i, TileRegs& r) __attribute__((always_inline)) -> uint32_t {  // returns its scales
    if ((i >> 6) != pg_at) {
      ask_pages(i >> 6, false);
      take_scales();
    }
    load_codes(i, r);
    return scales_at(i);
  };

  // ---- tiles in flight: kRing - 1 of the inner ones, and in front of them the first that has to be masked (the last of a
  //      sequence, for most calls): it is worked on first, while the others arrive
  constexpr int kRing = NQ == 1 ? 3 : 2;
  TileRegs ring[kRing];
  uint32_t sc[kRing];
  const int first_masked = in_lo > 0 ? 0 : in_hi;
  const int chunk = (first_masked < tiles ? first_masked : in_lo) >> 6;
  const bool near = (in_lo + kRing - 2) >> 6 == chunk;
  if (tiles > 0) {
    // (the first codes are asked for along with the scales, not behind them)
    ask_pages(chunk, early && chunk == 0);
    if (first_masked < tiles) load_codes(first_masked, ring[kRing - 1]);
#pragma unroll
    for (int r = 0; r < kRing - 1; ++r)
      if (near && in_lo + r < in_hi) load_codes(in_lo + r, ring[r]);
  }
  __builtin_amdgcn_sched_barrier(0);

  QFrag qf[NQ];
  f32x4 o[NQ][8];  // o[q][i][r]: query n of column q, element 32g + 8r + i
  float m_run[NQ], l_run[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    split_q(raw[q], qf[q]);
    m_run[q] = -INFINITY;
    l_run[q] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __builtin_amdgcn_sched_barrier(0);
  if (tiles > 0) {
    take_scales();
    sc[kRing - 1] = scales_at(first_masked);
#pragma unroll
    for (int r = 0; r < kRing - 1; ++r)
      if (in_lo + r < in_hi) sc[r] = near ? scales_at(in_lo + r) : load_tile(in_lo + r, ring[r]);
  }
  __builtin_amdgcn_sched_barrier(0);
  const float cs = a.p.softmax_scale * kLog2e;

  auto compute = [&](auto masked, int i, TileRegs& r, uint32_t sc) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked)::value;
    const int key0 = (t_first + stride * i) * kTileKeys;
    f32x4 st[2][NQ];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const i32x8 kf = {(int)r.k[hf][0][0], (int)r.k[hf][0][1], (int)r.k[hf][0][2], (int)r.k[hf][0][3],
                        (int)r.k[hf][1][0], (int)r.k[hf][1][1], (int)r.k[hf][1][2], (int)r.k[hf][1][3]};
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        st[hf][q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, qf[q].lo, z, 0, 0, 0, (int)(sc >> (8 * (hf % BLOCKS))), 0, qf[q].s_lo);
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        st[hf][q] =
            __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, qf[q].hi, st[hf][q], 0, 0, 0, (int)(sc >> (8 * (hf % BLOCKS))), 0, qf[q].s_hi);
    }
    bool has_nan = false;
    if constexpr (kMasked) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 16 * hf + 4 * g4 + e;
            if (key < my_lo[q] || key >= my_hi[q]) st[hf][q][e] = -INFINITY;
          }
        uint32_t any = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int key = key0 + 16 * hf + 4 * g4 + t;
          if (key < lo_first || key >= hi_last) r.v[hf][t] = u32x2{0u, 0u};  // seen by no row: whatever lies there
          any |= nan_bytes(r.v[hf][t][0]) | nan_bytes(r.v[hf][t][1]);
        }
        has_nan |= __builtin_amdgcn_ballot_w64(any != 0) != 0;
      }
    }
    const float ev[2] = {(float)((int)((sc >> 16) & 0xffu) - 127), (float)((int)(sc >> 24) - 127)};
    const float inv_v[2] = {__uint_as_float((254u - ((sc >> 16) & 0xffu)) << 23), __uint_as_float((254u - (sc >> 24)) << 23)};
    f16x8 pf[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      float mx[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const f32x4& v = st[hf][q];
        mx[hf] = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
      }
      const float top = quad_max(BLOCKS == 1 ? __builtin_fmaf(fmaxf(mx[0], mx[1]), cs, ev[0])
                                             : fmaxf(__builtin_fmaf(mx[0], cs, ev[0]), __builtin_fmaf(mx[1], cs, ev[1])));
      if (__builtin_amdgcn_ballot_w64(top > m_run[q]) != 0) {
        const float m_new = fmaxf(m_run[q], top);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[q] - m_new);
        m_run[q] = m_new;
        l_run[q] *= alpha;
#pragma unroll
        for (int i2 = 0; i2 < 8; ++i2)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[q][i2][e] *= alpha;
      }
      const float ref = m_run[q] == -INFINITY ? 0.f : m_run[q];
      u32x4 pw;
      float sum = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float off = ev[hf % BLOCKS] + kHeadroom - ref;
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[hf][q][e], cs, off));
          sum += w[e];
        }
        if (BLOCKS == 2 || hf == 1) {
          l_run[q] = __builtin_fmaf(sum, inv_v[hf % BLOCKS], l_run[q]);
          sum = 0.f;
        }
        pw[2 * hf] = pack_f16x2(w[0], w[1]);
        pw[2 * hf + 1] = pack_f16x2(w[2], w[3]);
      }
      pf[q] = __builtin_bit_cast(f16x8, pw);
    }
    if constexpr (kMasked) {
      if (__builtin_expect(has_nan, 0)) {
        f16x8 seen[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = key0 + 16 * (e >> 2) + 4 * g4 + (e & 3);
            seen[q][e] = key >= my_lo[q] && key < my_hi[q] ? (_Float16)1.f : (_Float16)0.f;
          }
#pragma unroll
        for (int i2 = 0; i2 < 8; ++i2) {
          f16x8 flag;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            flag[e] = (nan_bytes(r.v[e >> 2][e & 3][i2 >> 2]) >> (8 * (i2 & 3))) & 0x80u ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            const f32x4 z = {0.f, 0.f, 0.f, 0.f};
            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(flag, seen[q], z, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hit[e] > 0.f) o[q][i2][e] = NAN;
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t bad = nan_bytes(r.v[hf][t][w]);
              r.v[hf][t][w] &= ~((bad >> 7) * 0xffu);
            }
      }
    }
    // V^T: row n of M-tile 4w + e is element 8n + 4w + e.  Byte pairs of two tokens come together with one permute, and
    // the converter takes either half of it.
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t pr[2][2][2];  // [half][token pair][elements 01 | 23]
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          pr[hf][t][0] = __builtin_amdgcn_perm(r.v[hf][2 * t + 1][w], r.v[hf][2 * t][w], 0x05010400u);
          pr[hf][t][1] = __builtin_amdgcn_perm(r.v[hf][2 * t + 1][w], r.v[hf][2 * t][w], 0x07030602u);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f16x2 d[4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            d[2 * hf + t] = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(pr[hf][t][e >> 1], 1.0f, true)
                                  : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(pr[hf][t][e >> 1], 1.0f, false);
        const f16x8 vf = {d[0][0], d[0][1], d[1][0], d[1][1], d[2][0], d[2][1], d[3][0], d[3][1]};
#pragma unroll
        for (int q = 0; q < NQ; ++q)
          o[q][4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[q], o[q][4 * w + e], 0, 0, 0);
      }
    }
  };

  for (int i = first_masked; i < tiles;) {
    compute(std::true_type{}, i, ring[kRing - 1], sc[kRing - 1]);
    ++i;
    if (i == in_lo) i = in_hi;
    if (i < tiles) sc[kRing - 1] = load_tile(i, ring[kRing - 1]);
  }
  for (int i = in_lo; i < in_hi; i += kRing) {
#pragma unroll
    for (int r = 0; r < kRing; ++r) {
      constexpr int kLast = kRing - 1;
      if (i + r + kLast < in_hi) sc[(r + kLast) % kRing] = load_tile(i + r + kLast, ring[(r + kLast) % kRing]);
      if (i + r < in_hi) compute(std::false_type{}, i + r, ring[r], sc[r]);
    }
  }

  // ---- the waves' results join in LDS, one 16-row column at a time; half a wave then takes a row
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int lane = this_lane(), n16 = lane & 15, g4 = lane >> 4, d0 = (lane & 31) * 4;
    const int live = packed - pr0 - q * 16;  // rows behind the last one are worth no trip
    if (q) __syncthreads();
    const float l_row = quad_sum(l_run[q]);
    if (n16 < live) {
      if (g4 == 0) {
        sm->m[wave][n16] = m_run[q];
        sm->l[wave][n16] = l_row;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *reinterpret_cast<f32x4*>(&sm->o[wave][n16][32 * g4 + 8 * r + i]) =
              f32x4{o[q][i][r], o[q][i + 1][r], o[q][i + 2][r], o[q][i + 3][r]};
    }
    __syncthreads();
    static_assert(2 * kWaves == 16, "half a wave to a row");
    const int row16 = 2 * wave + (lane >> 5);
    if (row16 < live) {
      float m = -INFINITY, l = 0.f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sm->m[w][row16]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = join_factor(sm->m[w][row16], m);
        l = __builtin_fmaf(sm->l[w][row16], f, l);
        const f32x4 x = *reinterpret_cast<const f32x4*>(&sm->o[w][row16][d0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(x[e], f, acc[e]);
      }
      const int pr = pr0 + q * 16 + row16;
      if (piece >= 0) {
        const int64_t at = (int64_t)piece * (16 * NQ) + q * 16 + row16;
        *reinterpret_cast<f32x4*>(a.part_o + at * kKvDim + d0) = acc;
        if (d0 == 0) {
          a.part_ml[2 * at] = m;
          a.part_ml[2 * at + 1] = l;
        }
      } else {
        const float inv = s.ok ? (l == 0.f ? 0.f : 1.f / l) : NAN;
        const u32x2 w = {pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
        const int row = a.by_group(pr), hh = h * a.group + pr - row * a.group;
        *reinterpret_cast<u32x2*>((uint16_t*)a.p.out + times(s.row0 + row, a.p.o_sr) + times(hh, a.p.o_sh) + d0) = w;
      }
    }
  }
  }
}

// Joins the pieces of split key ranges: bound by its launch and two trips to memory, 3.5 us for 12 rows of 6 pieces, 5.2
// for 512 units of a shared-out call.  16 lanes x 8 elements read one piece of one packed query row; the 16 such groups
// of a workgroup take `ways` pieces of 16 / ways rows at once (ways: the number of pieces, up to a power of two and 16)
// and meet in LDS in a fixed order.  All pieces behind one another in a lane took 25 us for 26 of them.
__global__ __launch_bounds__(256) void kv_join_kernel(AttnArgs a, int ways_log2, Divisor by_blocks) {
  const int tid = threadIdx.x, grp = tid >> 4, d0 = (tid & 15) * 8;
  __shared__ float sm_o[16][kKvDim + 4];
  __shared__ float sm_m[16], sm_l[16];
  asm volatile("" ::"s"(a.n.row_start), "s"(a.p.out), "s"(a.p.total_rows), "s"(a.part_o));
  const int ways = 1 << ways_log2, per = 16 >> ways_log2, slot = grp >> ways_log2, way = grp & (ways - 1);
  const int blocks = (a.block_rows + per - 1) >> (4 - ways_log2);
  const int64_t cut = by_blocks(blockIdx.x);  // the unit, counted from the first that is cut
  const int r = (int)(blockIdx.x - cut * blocks) * per + slot;
  int b, h, qb;
  kv_unit(a, (uint32_t)(a.first_split + cut), b, h, qb);
  const KvSeq s = kv_seq(a.n, b, a.p.total_rows);
  const int pr = qb * a.block_rows + r;
  const bool live = r < a.block_rows && pr < s.rows * a.group;
  // Pieces of the unit: number t at piece0 + t * step, the first one place later.
  int pieces = a.splits, step = 1, odd = 0;
  int64_t piece0 = cut * a.splits;
  if (a.share) {
    const int lane = tid & 63;
    Lens lens;
    const int head_tiles = head_sum(a, lane, lens), total = head_tiles * a.c.heads;
    int first = h * head_tiles;
    for (int b0 = 0; b0 + 64 <= b; b0 += 64) {
      first += __builtin_amdgcn_readlane(lens.upto, 63);
      load_lens(a, b0 + 64, lane, lens);
    }
    const int count = __builtin_amdgcn_readlane(lens.count, b & 63);
    first += __builtin_amdgcn_readlane(lens.upto, b & 63) - count;
    pieces = 0;
    if (count > 0) {
      const int n = share_count(total, a.share);
      const int w0 = share_of(total, n, first), w1 = min(share_of(total, n, first + count - 1), n - 1);
      if (w0 == w1) return;  // one workgroup had all of it and wrote the result
      pieces = w1 - w0 + 1;  // the first workgroup's piece begins the unit, the others' continue it
      piece0 = 2 * (int64_t)w0;
      step = 2;
      odd = 1;
    }
  }
  float m = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int t = way; r < a.block_rows && t < pieces; t += ways) {  // (dead rows too: a piece has all of them)
    const int64_t at = (piece0 + (int64_t)t * step + (t == 0 ? odd : 0)) * a.block_rows + r;
    const float mt = a.part_ml[2 * at], lt = a.part_ml[2 * at + 1];
    const f32x4 lo = *reinterpret_cast<const f32x4*>(a.part_o + at * kKvDim + d0);
    const f32x4 hi = *reinterpret_cast<const f32x4*>(a.part_o + at * kKvDim + d0 + 4);
    const float mn = fmaxf(m, mt);
    const float fo = join_factor(m, mn), fn = join_factor(mt, mn);
    m = mn;
    l = l * fo + lt * fn;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] = acc[e] * fo + lo[e] * fn;
      acc[4 + e] = acc[4 + e] * fo + hi[e] * fn;
    }
  }
  if (ways > 1) {
    *reinterpret_cast<f32x4*>(&sm_o[grp][d0]) = f32x4{acc[0], acc[1], acc[2], acc[3]};
    *reinterpret_cast<f32x4*>(&sm_o[grp][d0 + 4]) = f32x4{acc[4], acc[5], acc[6], acc[7]};
    if (d0 == 0) {
      sm_m[grp] = m;
      sm_l[grp] = l;
    }
    __syncthreads();
    if (way != 0) return;
    for (int g = grp + 1; g < grp + ways; ++g) m = fmaxf(m, sm_m[g]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int g = grp; g < grp + ways; ++g) {
      const float f = join_factor(sm_m[g], m);
      l = __builtin_fmaf(sm_l[g], f, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(sm_o[g][d0 + e], f, acc[e]);
    }
  }
  if (!live) return;
  const float inv = s.ok ? (l == 0.f ? 0.f : 1.f / l) : NAN;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  const int row = a.by_group(pr), hh = h * a.group + pr - row * a.group;
  *reinterpret_cast<u32x4*>((uint16_t*)a.p.out + times(s.row0 + row, a.p.o_sr) + times(hh, a.p.o_sh) + d0) = w;
}

struct Plan {
  int nq;  // 16-row columns of the streaming form; 0: the tile form
  int block_rows, nqb, share, splits, ways, ways_log2;
  int64_t units, first_split, join_units, ws_bytes;
};

int check(const dsx_kv_cache* c, const dsx_kv_batch* n, const dsx_kv_attn_params* p) {
  if (!p) return DSX_ENULL;
  const int rc = kv_check_cache(c, n, p->total_rows);
  if (rc != DSX_OK) return rc;
  if (p->heads_q < 1 || p->heads_q % c->heads || p->window < 0) return DSX_EBADSHAPE;
  if (!(p->softmax_scale > 0.f) || !(p->softmax_scale * kLog2e < INFINITY)) return DSX_EBADSHAPE;
  if ((int64_t)n->max_rows * (p->heads_q / c->heads) > (1 << 30)) return DSX_EBADSHAPE;
  return DSX_OK;
}

Plan make_plan(const dsx_kv_cache& c, const dsx_kv_batch& n, const dsx_kv_attn_params& p) {
  Plan r{};
  const int64_t rows = n.max_rows < p.total_rows ? n.max_rows : p.total_rows;
  const int64_t packed = rows * (p.heads_q / c.heads);
  const int64_t span = p.window > 0 && p.window + rows < n.max_kv_len ? p.window + rows : n.max_kv_len;
  int cus = device_cus();
  if (cus <= 0) cus = 256;
  // Up to 16 rows are one column of the matrix instruction.  More go to the streaming form in blocks of two columns when
  //  * one block has them all, or
  //  * two do and no compute unit gets two blocks (16 x 40 rows, 8 heads, 1024 tokens: 17.5 us against the tile form's 29.2;
  //    8 x 5, group 7, window 4096: 23 against 29) or the cache is long (24 x 9, group 4, 8192 tokens: 127 against 168 us;
  //    64 x 8, group 5, 4096: 145 against 152; but 2048: 94 against 87, 512: 47 against 35), or
  //  * any number does, no compute unit gets two, and either there are two for each block, so that it can be cut (1 x 160
  //    rows, 12 heads, 8192 tokens: 29 against 38), or the cache is short (1 x 600, 12 heads, 2048 tokens: 25 against 41 us,
  //    512: 14 against 25; 4 x 40, group 7, 3900: 36 against 43; but 1 x 100, 40 heads, 16384: 114 against 80).
  // The rest is the tile form's, which loads a key once for 256 rows: at two blocks a compute unit it wins or draws (1 x
  // 390, 30 heads, 2048 tokens: 42 against 43; 3900: 54 against 66).
  // All of this was measured on batches whose sequences have about as many rows each: the rule knows only the most.  4096
  // rows over 4096 tokens and 63 x 1 over 16384, 32 / 8 heads: 2250 us in one call, all of it in the tile form, 146 and 296
  // in two; 64 over 16384 and 63 x 1: 626 against 42 + 297.
  const int64_t blocks = (packed + 31) / 32, wgs = blocks * n.batch * c.heads;
  const bool one_each = wgs <= cus, long_cache = span >= 4096;
  const bool stream = blocks <= 1   ? true
                      : blocks == 2 ? one_each || long_cache
                                    : one_each && (2 * wgs <= cus || !long_cache);
  r.nq = packed <= 16 ? 1 : stream ? 2 : 0;
  r.block_rows = r.nq ? 16 * r.nq : kTileRows;
  r.nqb = (int)((packed + r.block_rows - 1) / r.block_rows);
  r.units = (int64_t)n.batch * c.heads * r.nqb;
  r.splits = 1;
  r.first_split = r.units;
  r.ways = 1;
  int64_t pieces = 0;
  if (r.nq) {
    const int64_t tiles = (span + kTileKeys - 1) / kTileKeys + 1;
    // The longest a compute unit's share can be, in tiles.  From 512 on, even shares and a join (which costs 5 us) beat one
    // workgroup per unit and its uneven end: 64 x 16384 tokens, 8 heads (1024 tiles): 280 against 305 us; 32 x 16384 (512):
    // 168 against 178; 32 x 8192 (256): 93 against 86; 32 x 4097 (129): 58 against 44.
    // Fewer units than compute units are cut into equal pieces, as many as there are compute units and tiles for the waves,
    // from four tiles a wave on: replayed from a graph, 1 x 1561 tokens, 12 heads (six pieces): 10.1 against 13.1 us, 1000
    // tokens: 9.2 against 10.7, 4 x 5 rows, 4 heads, 1000 tokens: 13.5 against 14.7; below that the join costs more than it
    // saves (cut at 800 tokens: 15.4 against 14.9, at 500: 14.0 against 12.6, before later steps).  Fewer, longer pieces
    // bring nothing (1561 tokens in three: 12.7 against 11.6, at the same time).
    const int64_t load = r.units * tiles / cus;
    if (load >= 512 && r.nqb == 1 && r.units * tiles < (1ll << 30)) {
      r.share = cus;
      pieces = 2 * (int64_t)r.share;
      r.ways = (int)((r.share + r.units - 1) / r.units) + 1;
    } else if (r.units < cus && r.units > 0 && tiles >= 4 * kWaves) {
      r.splits = (int)std::min<int64_t>(cus / r.units, tiles / kWaves);
      if (r.splits > 1) pieces = r.units * r.splits;
      r.ways = r.splits;
    }
    if (pieces > 0) {
      r.first_split = 0;
      r.join_units = r.units;
    }
  } else {
    int64_t tail;
    kv_tile_split(r.units, span, cus, tail, r.splits);
    r.first_split = r.units - tail;
    pieces = tail * r.splits;
    r.join_units = tail;
    r.ways = r.splits;
  }
  while ((1 << r.ways_log2) < r.ways && r.ways_log2 < 4) ++r.ways_log2;
  r.ws_bytes = pieces * r.block_rows * (kKvDim + 2) * 4;
  return r;
}

template <int NQ, int BLOCKS, bool SHARE>
int launch_stream(const AttnArgs& a, unsigned workgroups, hipStream_t st) {
  static PerDeviceOnce attr_once;
  const int rc = per_device_once(attr_once, [](int) {
    return hipFuncSetAttribute((const void*)kv_stream_kernel<NQ, BLOCKS, SHARE>, hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)sizeof(StreamLds)) == hipSuccess ? (int)DSX_OK : (int)DSX_ELAUNCH;
  });
  if (rc != DSX_OK) return rc;
  kv_stream_kernel<NQ, BLOCKS, SHARE><<<dim3(workgroups), dim3(64 * kWaves), sizeof(StreamLds), st>>>(a);
  return DSX_OK;
}
template <int NQ, int BLOCKS>
int launch_stream(const AttnArgs& a, int64_t units, hipStream_t st) {
  return a.share ? launch_stream<NQ, BLOCKS, true>(a, (unsigned)a.share, st)
                 : launch_stream<NQ, BLOCKS, false>(a, (unsigned)(units * a.splits), st);
}
template <int NQ>
int launch_stream(const AttnArgs& a, int64_t units, hipStream_t st) {
  return a.c.page_size >= kTileKeys ? launch_stream<NQ, 1>(a, units, st) : launch_stream<NQ, 2>(a, units, st);
}

}  // namespace
}  // namespace dsx

extern "C" int64_t dsx_kv_attn_workspace_bytes(const dsx_kv_cache* cache, const dsx_kv_batch* batch,
                                               const dsx_kv_attn_params* p) {
  using namespace dsx;
  if (check(cache, batch, p) != DSX_OK) return 0;
  return make_plan(*cache, *batch, *p).ws_bytes;
}

extern "C" int dsx_kv_attn(const dsx_kv_cache* cache, const dsx_kv_batch* batch, const dsx_kv_attn_params* p,
                           void* stream) {
  using namespace dsx;
  const int rc = check(cache, batch, p);
  if (rc != DSX_OK) return rc;
  const dsx_kv_cache& c = *cache;
  const dsx_kv_batch& n = *batch;
  if (!p->q || !p->out) return DSX_ENULL;
  if (!kv_rows_ok(p->q, p->q_sr, p->q_sh) || !kv_rows_ok(p->out, p->o_sr, p->o_sh) || ((uintptr_t)p->workspace & 15))
    return DSX_EALIGN;
  if (n.max_rows == 0 || p->total_rows == 0) return DSX_OK;
  Plan plan = make_plan(c, n, *p);
  if (plan.ws_bytes > 0) {
    if (!p->workspace) {
      plan.splits = 1;
      plan.share = 0;
      plan.first_split = plan.units;
      plan.join_units = 0;
    } else if (p->workspace_bytes < plan.ws_bytes) {
      return DSX_EWORKSPACE;
    }
  }
  const int per = 16 >> plan.ways_log2, join_blocks = (plan.block_rows + per - 1) / per;
  const int64_t join_wgs = plan.join_units * join_blocks;
  // A launch has fewer than 2^32 threads: 512 a unit (and a few more where the tile form cuts some), 256 a join.
  if (plan.units >= (1ll << 23) - 4096 || join_wgs >= (1ll << 24)) return DSX_EBADSHAPE;
  AttnArgs a{};
  a.c = c;
  a.n = n;
  a.p = *p;
  a.group = p->heads_q / c.heads;
  a.page_shift = __builtin_ctz((unsigned)c.page_size);
  a.block_rows = plan.block_rows;
  a.nqb = plan.nqb;
  a.share = plan.share;
  a.splits = plan.splits;
  a.first_split = plan.first_split;
  a.by_group = Divisor::of(a.group);
  a.by_nqb = Divisor::of(a.nqb);
  a.by_batch = Divisor::of(n.batch);
  a.by_splits = Divisor::of(a.splits);
  if (plan.join_units > 0) {
    a.part_o = (float*)p->workspace;
    a.part_ml = a.part_o + plan.ws_bytes / (4 * (kKvDim + 2)) * kKvDim;
  }
  hipStream_t st = (hipStream_t)stream;
  const int lrc = plan.nq == 1   ? launch_stream<1>(a, plan.units, st)
                  : plan.nq == 2 ? launch_stream<2>(a, plan.units, st)
                                 : launch_kv_tile(a, plan.units, st);
  if (lrc != DSX_OK) return lrc;
  if (hipGetLastError() != hipSuccess) return DSX_ELAUNCH;
  if (join_wgs > 0)
    kv_join_kernel<<<dim3((unsigned)join_wgs), dim3(256), 0, st>>>(a, plan.ways_log2, Divisor::of(join_blocks));
  return hipGetLastError() == hipSuccess ? DSX_OK : DSX_ELAUNCH;
}
