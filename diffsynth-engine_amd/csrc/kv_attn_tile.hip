// Attention over the paged 8-bit key/value cache, the form for many query rows.  Mathematics, operand formats and unit
// numbering as in kv_attn.hip; here a workgroup's 256 query rows share every key that is loaded and every V code that is
// converted.
//
// One workgroup = 8 waves x 32 query rows (two 16-row MFMA columns each), one per compute unit.  Tiles of 64 keys:
//  * K and V codes go memory -> LDS with global_load_lds_dwordx4, 16 KiB a tile, four stages, three tiles ahead.  K stays
//    8 bits wide all the way into the matrix instruction: half the LDS traffic of a 16-bit K.
//  * V is transposed and widened to fp16 once per workgroup and tile (each wave an eighth: four 4-byte reads, four byte
//    permutes, eight conversions, four 8-byte writes) into a second LDS buffer that holds operand fragments as they are
//    read, lane after lane.
//  * Interval kb, behind one barrier: S(kb+1)^T = K Q^T (16 MFMAs) with the rest of the exponentials of tile kb and the
//    conversion of V(kb+1) between them, then O^T += V(kb)^T P(kb)^T (32 MFMAs) with the maximum of S(kb+1) and its first
//    exponentials.  Two waves share a SIMD; without the interleaving both would do matrix and vector work in step.
//  * The running maximum is a reference that moves only when it has to: weights are exp2(s c + e_v + 8 - m), and only when
//    some of them would leave fp16 (2^15) does m become the maximum so far.  A tile that does not move it costs no
//    rescaling of O, and where a tile has one scale (pages of 64 and more) no look at its scores' maximum either: the row
//    sums, which are needed anyway, tell.
// Bound: the matrix pipe with the vector work and LDS beside it: 2050 cycles of matrix instructions a tile and SIMD, 1960 of
// vector issue, 1170 of LDS reads and writes, by counters; 3380 measured over 512 tiles (at 1.85 of 2.4 GHz in that run).
// 4680 rows over 32760 tokens, 40 heads: 2.41 to 2.57 ms by machine, 1222 to 1303 TFLOP/s of the two products (a large bf16
// matrix product: 1525; the framework's attention over bf16 keys of the same size: 1125 to 1250); pages of 16: 2.67 ms
// (236 vector instructions a wave and tile instead of 194).  3 prompts of 4096 rows, 37 tiles a unit: 0.325 ms and 3980 cycles
// a tile, with its share of the units' beginnings and ends.  On the
// first case (2.65 ms then), in copies with work left out: without q's low term 8 % less, without exponentials 4 %, without
// V's conversion 5 %, without the scores' maximum 7 % (of which looking at the row sums instead got 5).  Exponentials in
// other places (two to six in front of the first product, 8 to 20 in the second stage), three or four fragments of V ahead:
// no change beyond noise.
// LDS: K and V rows are 128 bytes; 16-byte piece j of K row r lies at j ^ (r & 7) (the permutation is applied to the
// source address, the destination of a direct load being linear).
#include "kv_attn_internal.h"

namespace dsx {
namespace {

constexpr int KB = 64;
constexpr int kRaw = KB * kKvDim;          // 8 KiB: one tile of K or of V
constexpr int kStages = 4;
constexpr int kVf = kRaw * 2;              // 16 KiB: one tile of V in fp16 fragments
constexpr int kOffV = kStages * kRaw, kOffVf = 2 * kStages * kRaw, kOffFlag = kOffVf + 2 * kVf;
constexpr int kLdsBytes = kOffFlag + 2 * 8 * 4;
constexpr float kTileHeadroom = 8.f;       // log2 of a weight at the reference
constexpr float kMoveAt = 7.f;             // the reference moves when a score is further above it: 8 + 7 < 16 (fp16)
constexpr float kMostSum = 32768.f;        // a lane's weights of one tile
constexpr float kNoRef = -3.0e38f;         // reference of a row that has seen no token: finite, so that -inf stays -inf

typedef __attribute__((address_space(3))) void* lptr_t;

// Largest of three (fmaxf twice would canonicalise its operands first).  Reads matrix results: behind mfma_settle.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm volatile("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}
// The wait states between a matrix instruction and inline assembly that reads its result, which the compiler does not
// see: 11 for the eight passes of the 16x16x128 shape.
__device__ __forceinline__ void mfma_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 11" ::: "memory");
}

// UNI: pages of 64 tokens or more, so that a tile lies in one block and has one scale of K and one of V; otherwise every
// 16-key group has its own.
template <bool UNI>
__global__ __launch_bounds__(512, 2) void kv_tile_kernel(AttnArgs a, int64_t units, int whole8, int cut8) {
  constexpr int kGroups = UNI ? 1 : 4;  // scales of a tile
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const dsx_kv_cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, n16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups are dealt round-robin to the eight XCDs: each XCD takes a contiguous run of units, so that the query
  // blocks of one head find its keys in one L2.  Whole units first, then the pieces of the units that are cut.
  int64_t unit;
  int split = 0, splits = 1;
  if ((int)blockIdx.x < whole8) {
    unit = (int64_t)(blockIdx.x & 7) * (whole8 >> 3) + (blockIdx.x >> 3);
    if (unit >= a.first_split) return;
  } else {
    const unsigned j = blockIdx.x - whole8;
    const unsigned piece = (j & 7) * (unsigned)(cut8 >> 3) + (j >> 3);
    if (piece >= (units - a.first_split) * a.splits) return;
    const unsigned cut = a.by_splits(piece);
    unit = a.first_split + cut;
    split = (int)(piece - cut * a.splits);
    splits = a.splits;
  }
  int b, h, qb;
  kv_unit(a, (uint32_t)unit, b, h, qb);
  b = __builtin_amdgcn_readfirstlane(b);
  h = __builtin_amdgcn_readfirstlane(h);
  qb = __builtin_amdgcn_readfirstlane(qb);
  KvSeq s = kv_seq(a.n, b, a.p.total_rows);
  s.rows = __builtin_amdgcn_readfirstlane(s.rows);
  s.kv = __builtin_amdgcn_readfirstlane(s.kv);
  const int packed = s.rows * a.group;
  const int pr0 = qb * kTileRows;
  if (pr0 >= packed) return;

  // ---- spans: of the workgroup (first and last row), of the wave, of the lane's two rows
  const int causal = a.p.causal, window = a.p.window;
  int lo_first, hi_first, lo_last, hi_last, wlo_first, whi_first, wlo_last, whi_last;
  kv_row_span(s.kv, s.rows, a.by_group(pr0), causal, window, lo_first, hi_first);
  kv_row_span(s.kv, s.rows, a.by_group(min(pr0 + kTileRows, packed) - 1), causal, window, lo_last, hi_last);
  const int wr0 = pr0 + wave * 32;
  const bool active = wr0 < packed;
  kv_row_span(s.kv, s.rows, a.by_group(min(wr0, packed - 1)), causal, window, wlo_first, whi_first);
  kv_row_span(s.kv, s.rows, a.by_group(min(wr0 + 31, packed - 1)), causal, window, wlo_last, whi_last);
  const int tile_first = lo_first / KB, tile_last = (hi_last + KB - 1) / KB;
  const int per = (max(tile_last - tile_first, 0) + splits - 1) / splits;
  const int kb_begin = tile_first + split * per;
  const int kb_end = min(kb_begin + per, tile_last);

  QFrag qf[2];
  int my_lo[2];
  uint32_t my_n[2];  // tokens that the row sees, from my_lo on
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    int end;
    QRaw raw;
    load_q(a, s, h, min(wr0 + 16 * t + n16, packed - 1), g4, raw, my_lo[t], end);
    split_q(raw, qf[t]);
    my_n[t] = (uint32_t)(end - my_lo[t]);
  }

  f32x4 o[8][2];  // o[i][t][r]: row n of column t, element 32g + 8r + i
  float m_ref[2] = {kNoRef, kNoRef}, l_run[2] = {0.f, 0.f}, lsum[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) o[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (kb_begin < kb_end) {
    const float cs = a.p.softmax_scale * kLog2e;
    const uint8_t* kbase = (const uint8_t*)c.k + (int64_t)h * c.k_sh;
    const uint8_t* vbase = (const uint8_t*)c.v + (int64_t)h * c.v_sh;
    const int page_mask = c.page_size - 1;

    // Page numbers of the wave's eight keys of a tile, and the scales of a tile's 16-key groups: 64 tiles ahead at once,
    // one tile per lane.  Tiles and keys beyond the end take the last key's page: their codes are loaded and not used.
    int pg = 0, pg_at = -64;
    auto page_of = [&](int kb) __attribute__((always_inline)) -> int {
      const int i = kb - kb_begin;
      if (__builtin_expect(i - pg_at >= 64, 0)) {
        const AttnArgs& r = args_again();
        pg_at = i & ~63;
        const int id = r.n.page_table[times(b, r.n.table_sb) +
                                      (min((kb_begin + pg_at + lane) * KB + 8 * wave, hi_last - 1) >> r.page_shift)];
        pg = id < 0 || id >= r.c.pages ? 0 : id;
      }
      return __builtin_amdgcn_readlane(pg, i & 63);
    };
    uint32_t ks_all = 0, vs_all = 0;
    int sc_at = -64;
    auto scales_of = [&](int kb, uint32_t& ks, uint32_t& vs) __attribute__((always_inline)) {
      const int i = kb - kb_begin;
      if (__builtin_expect(i - sc_at >= 64, 0)) {
        const AttnArgs& r = args_again();
        sc_at = i & ~63;
        ks_all = vs_all = 0;
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          const int id = r.n.page_table[times(b, r.n.table_sb) +
                                        (min((kb_begin + sc_at + lane) * KB + 16 * q, hi_last - 1) >> r.page_shift)];
          const bool bad = id < 0 || id >= r.c.pages;
          const int page = bad ? 0 : id;
          uint32_t k8 = ((const uint8_t*)r.c.k_scale)[times(page, r.c.ks_sp) + h];
          uint32_t v8 = ((const uint8_t*)r.c.v_scale)[times(page, r.c.vs_sp) + h];
          if (bad || v8 == 255) {  // NaN scores for every row that sees the block, and nothing for the others
            k8 = 255;
            v8 = 127;
          }
          ks_all |= k8 << (8 * q);
          vs_all |= v8 << (8 * q);
        }
      }
      ks = (uint32_t)__builtin_amdgcn_readlane((int)ks_all, i & 63);
      vs = (uint32_t)__builtin_amdgcn_readlane((int)vs_all, i & 63);
    };

    // ---- direct loads: one wave instruction = 1 KiB = 8 keys.  Inline assembly, so that the compiler does not put a
    //      wait for them in front of every LDS read; vmcnt waits and barriers below order them.
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)smem;
    const uint32_t off_v = (uint32_t)(lane * 16);
    const uint32_t off_k = (uint32_t)((lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    auto dma16 = [&](const uint8_t* base, uint32_t off, uint32_t lds_addr) {
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                   :
                   : "v"(off), "s"(base), "s"(lds_addr)
                   : "memory", "m0");
    };
#pragma clang diagnostic pop
    int64_t src = 0;  // page and token offset of the tile that is issued, in tokens of a block
    int src_page = 0;
    auto aim = [&](int kb) {  // the tile that the next two loads fetch (the last one again beyond the end: nobody reads it)
      kb = min(kb, kb_end - 1);
      src_page = page_of(kb);
      src = (int64_t)((kb * KB + 8 * wave) & page_mask) * kKvDim;
    };
    auto issue_k = [&](int stage) {
      dma16(kbase + times(src_page, c.k_sp) + src, off_k, lds0 + stage * kRaw + wave * 1024);
    };
    auto issue_v = [&](int stage) {
      dma16(vbase + times(src_page, c.v_sp) + src, off_v, lds0 + kOffV + stage * kRaw + wave * 1024);
    };

    // Some row of the workgroup does not see some key of the tile.
    auto boundary = [&](int kb) { return kb * KB < lo_last || (kb + 1) * KB > hi_first; };

    // ---- V: raw tile -> fp16 fragments.  Wave: 32-key chunk wave / 4, byte half (wave / 2) % 2 of every 8-element group,
    //      16-key half wave % 2.  Fragment (chunk, i), lane (n, g): element 8n + i of keys 4g .. 4g + 3 of both halves.
    const int cv_ch = wave >> 2, cv_w = (wave >> 1) & 1, cv_hf = wave & 1;
    const int cv_src = kOffV + (32 * cv_ch + 16 * cv_hf + 4 * g4) * kKvDim + 8 * n16 + 4 * cv_w;
    const int cv_dst = kOffVf + (cv_ch * 8 + 4 * cv_w) * 1024 + lane * 16 + cv_hf * 8;
    auto cv_read = [&](int stage, uint32_t (&r)[4]) {
#pragma unroll
      for (int t = 0; t < 4; ++t) r[t] = *reinterpret_cast<const uint32_t*>(smem + cv_src + stage * kRaw + t * kKvDim);
    };
    // A boundary tile: tokens that no row sees may be anything and become 0; NaN of the others becomes 0 too, because it
    // must not reach (as 0 * NaN) the rows that do not see it, and is handed to the others by nan_rows.
    auto cv_fix = [&](int kb, int buf, uint32_t (&r)[4]) {
      uint32_t any = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int key = kb * KB + 32 * cv_ch + 16 * cv_hf + 4 * g4 + t;
        if (key < lo_first || key >= hi_last) r[t] = 0;
        const uint32_t bad = nan_bytes(r[t]);
        r[t] &= ~((bad >> 7) * 0xffu);
        any |= bad;
      }
      const bool found = __builtin_amdgcn_ballot_w64(any != 0) != 0;
      if (lane == 0) *reinterpret_cast<int*>(smem + kOffFlag + (buf * 8 + wave) * 4) = found;
    };
    auto cv_write = [&](int buf, const uint32_t (&r)[4]) {
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {  // elements 2 e2, 2 e2 + 1
        const uint32_t sel = e2 ? 0x07030602u : 0x05010400u;
        const uint32_t p0 = __builtin_amdgcn_perm(r[1], r[0], sel), p1 = __builtin_amdgcn_perm(r[3], r[2], sel);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f16x2 d0, d1;
          if (e) {
            d0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p0, 1.0f, true);
            d1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p1, 1.0f, true);
          } else {
            d0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p0, 1.0f, false);
            d1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(p1, 1.0f, false);
          }
          const u32x2 w = {__builtin_bit_cast(uint32_t, d0), __builtin_bit_cast(uint32_t, d1)};
          *reinterpret_cast<u32x2*>(smem + cv_dst + buf * kVf + (2 * e2 + e) * 1024) = w;
        }
      }
    };

    // ---- operands
    const int lane_k = n16 * kKvDim + ((g4 ^ (n16 & 7)) << 4);
    auto k_frag = [&](int stage, int q) {  // keys 16q .. 16q + 15
      const u32x4 x = *reinterpret_cast<const u32x4*>(smem + stage * kRaw + q * 2048 + lane_k);
      const u32x4 y = *reinterpret_cast<const u32x4*>(smem + stage * kRaw + q * 2048 + (lane_k ^ 64));
      return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    };
    // (one base for all of them: the offsets from the start of LDS are too long for the instruction's field, and each would
    // be a sum of its own)
    int lane_v = kOffVf + lane * 16;
    asm volatile("" : "+v"(lane_v));
    auto v_frag = [&](int buf, int f) { return *reinterpret_cast<const f16x8*>(smem + lane_v + (buf * kVf + f * 1024)); };
#define DSX_QK(KF, Q, T, PART, ACC) \
  __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(KF, qf[T].PART, ACC, 0, 0, UNI ? 0 : Q, (int)ks, 0, qf[T].s_##PART)
    const f32x4 zero4 = {0.f, 0.f, 0.f, 0.f};

    // Position of the tile's key 4g in the row's span.  (Opaque: the differences of all 64 keys would be taken out of the
    // loop, into registers that it needs.)
    auto span_at = [&](int kb, int t) __attribute__((always_inline)) {
      int at = kb * KB + 4 * g4 - my_lo[t];
      asm volatile("" : "+v"(at));
      return at;
    };
    auto mask = [&](f32x4 (&st)[4][2], int kb) __attribute__((always_inline)) {
      if (__builtin_expect(kb * KB < wlo_last || (kb + 1) * KB > whi_first, 0)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int at = span_at(kb, t);
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = st[q][t][e];
              x = (uint32_t)(at + 16 * q + e) >= my_n[t] ? -INFINITY : x;
              asm volatile("" : "+v"(x));  // (one condition at a time: all of them at once are kept in scalar registers)
              st[q][t][e] = x;
            }
        }
      }
    };
    // Largest s c + e_v of the lane's own keys for its two rows: a quarter of each row.
    auto scan = [&](const f32x4 (&st)[4][2], const float (&ev)[kGroups], float (&mx)[2]) __attribute__((always_inline)) {
      mfma_settle();
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (UNI) {
          float x = max3(st[0][t][0], st[0][t][1], st[0][t][2]), y = max3(st[1][t][0], st[1][t][1], st[1][t][2]);
          x = max3(x, st[0][t][3], st[2][t][0]);
          y = max3(y, st[1][t][3], st[3][t][0]);
          x = max3(x, st[2][t][1], st[2][t][2]);
          y = max3(y, st[3][t][1], st[3][t][2]);
          x = max3(x, st[2][t][3], st[3][t][3]);
          mx[t] = __builtin_fmaf(max3(x, y, y), cs, ev[0]);
        } else {
          float x[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float y = max3(st[q][t][0], st[q][t][1], st[q][t][2]);
            x[q] = __builtin_fmaf(max3(y, y, st[q][t][3]), cs, ev[q]);
          }
          const float y = max3(x[0], x[1], x[2]);
          mx[t] = max3(y, y, x[3]);
        }
      }
    };
    auto must_move = [&](const float (&mx)[2]) {
      return __builtin_amdgcn_ballot_w64(mx[0] - m_ref[0] > kMoveAt || mx[1] - m_ref[1] > kMoveAt) != 0;
    };
    // New references for the wave's rows; O, the row sums and the weights `pw` that are still to be multiplied follow.
    // (Weights that were rounded to fp16 are rounded again, 2^-10 in all: making them anew would take their scores' registers,
    // which hold the next tile's by then.  Once at most, a tile's weights being used up in the same interval.)
    auto move = [&](const float (&mx)[2], uint32_t (&pw)[2][2][4], bool with_pw) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float to = fmaxf(m_ref[t], quad_max(mx[t]));
        const float alpha = __builtin_amdgcn_exp2f(m_ref[t] - to);
        m_ref[t] = to;
        l_run[t] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][t][e] *= alpha;
        if (with_pw) {
#pragma unroll
          for (int ch = 0; ch < 2; ++ch)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const f16x2 x = __builtin_bit_cast(f16x2, pw[ch][t][w]);
              pw[ch][t][w] = pack_f16x2((float)x[0] * alpha, (float)x[1] * alpha);
            }
        }
      }
    };
    auto scale_floats = [&](uint32_t vs, float (&ev)[kGroups], float (&inv)[kGroups]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < kGroups; ++q) {
        const uint32_t x = (vs >> (8 * q)) & 0xffu;
        ev[q] = (float)((int)x - 127);
        inv[q] = __uint_as_float((254u - x) << 23);
      }
    };
    // Entry n (0..31) of P = exp2(S c + off), in the order the second product takes them: 32-key chunk n / 16, column
    // (n / 8) % 2, word (n / 2) % 4, half n % 2.  The empty asm pins each result where it is computed, between the MFMAs
    // it is written beside; the optimiser would sink it to its first use.
    float p_even = 0.f;
    auto exp_entry = [&](const f32x4 (&st)[4][2], const float (&off)[kGroups][2], const float (&inv)[kGroups],
                         uint32_t (&pw)[2][2][4], int n) __attribute__((always_inline)) {
      const int ch = n >> 4, t = (n >> 3) & 1, w = (n >> 1) & 3, q = 2 * ch + (w >> 1);
      float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(st[q][t][2 * (w & 1) + (n & 1)], cs, off[UNI ? 0 : q][t]));
      lsum[t] = UNI ? lsum[t] + pv : __builtin_fmaf(pv, inv[q], lsum[t]);
      if (n & 1) {
        uint32_t word = pack_f16x2(p_even, pv);
        asm volatile("" : "+v"(word), "+v"(lsum[t]));
        pw[ch][t][w] = word;
      } else {
        asm volatile("" : "+v"(pv), "+v"(lsum[t]));
        p_even = pv;
      }
    };
    auto offsets = [&](const float (&ev)[kGroups], float (&off)[kGroups][2]) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < kGroups; ++q)
#pragma unroll
        for (int t = 0; t < 2; ++t) off[q][t] = ev[q] + kTileHeadroom - m_ref[t];
    };

    // NaN among the V codes of a boundary tile: NaN for the rows that see one, element by element, from the raw tile (its
    // stage is not filled again before the next interval).
    auto nan_rows = [&](int kb, int buf, int stage) __attribute__((always_inline)) {
      const int flag = *reinterpret_cast<const int*>(smem + kOffFlag + (buf * 8 + (lane & 7)) * 4);
      if (__builtin_amdgcn_ballot_w64(flag != 0) == 0) return;
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        f16x8 seen[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int at = span_at(kb, t);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            seen[t][e] = (uint32_t)(at + 32 * ch + 16 * (e >> 2) + (e & 3)) < my_n[t] ? (_Float16)1.f : (_Float16)0.f;
        }
        int codes = kOffV + stage * kRaw + (32 * ch + 4 * g4) * kKvDim + 8 * n16;
        asm volatile("" : "+v"(codes));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f16x8 bad;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            bad[e] = (smem[codes + (16 * (e >> 2) + (e & 3)) * kKvDim + i] & 0x7f) == 0x7f ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, seen[t], zero4, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = o[i][t][e];
              x = hit[e] > 0.f ? NAN : x;
              asm volatile("" : "+v"(x));
              o[i][t][e] = x;
            }
          }
        }
      }
    };

    constexpr int kExpEarly = 12;  // entries of P(kb + 1) made in stage 2 of interval kb; even
    constexpr int kScanFrags = 4;  // V fragments in front of the look at S(kb + 1)
    static_assert(32 - kExpEarly <= 32 && kExpEarly <= 2 * (16 - kScanFrags), "every entry has a slot");
    constexpr int kAhead = 2;      // V fragments read ahead of their MFMAs

#define DSX_HEAD(N) asm volatile("s_waitcnt vmcnt(" #N ") lgkmcnt(0)\n\ts_barrier" ::: "memory")

    f32x4 sA[4][2], sB[4][2];
    uint32_t pwA[2][2][4], pwB[2][2][4];
    float offA[kGroups][2], offB[kGroups][2], invA[kGroups], invB[kGroups];

    uint32_t ks, vs;  // scales of tile kb + 1
    auto interval = [&](int kb, int buf, f32x4 (&s_cur)[4][2], f32x4 (&s_next)[4][2], uint32_t (&pw_cur)[2][2][4],
                        uint32_t (&pw_next)[2][2][4], float (&off_cur)[kGroups][2],
                        const float (&inv_cur)[kGroups], float (&off_next)[kGroups][2], float (&inv_next)[kGroups]) __attribute__((always_inline)) {
      const int i = kb - kb_begin;
      const int st1 = (i + 1) & 3, st3 = (i + 3) & 3;
      const bool more = kb + 1 < kb_end;
      DSX_HEAD(2);  // tile kb + 1 has landed, the fragments of V(kb) are written
      // The two waves of a SIMD come here together, and of equal ones the first goes first: it was 900 of 3850 cycles early
      // at the next barrier.  So the second leads in the first stage, and the first in the second.
      if (wave >= 4) __builtin_amdgcn_s_setprio(1);
      {
        // ---- stage 1
        uint32_t raw[4];
        cv_read(st1, raw);
        if (__builtin_expect(boundary(kb + 1), 0)) cv_fix(kb + 1, buf ^ 1, raw);
        i32x8 kf[2] = {k_frag(st1, 0), k_frag(st1, 1)};
        f16x8 vf[kAhead + 1];
        int n = kExpEarly;
        // Two 16-key groups at a time: their low terms for both columns, then their high terms, so that none waits for the
        // product that it adds to.
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int q = 2 * (x >> 3) + ((x >> 1) & 1), col = x & 1;
          const bool high = (x >> 2) & 1;
#define DSX_STEP(Q, T)                                                            \
  if (q == Q && col == T) {                                                       \
    if (high)                                                                     \
      s_next[Q][T] = DSX_QK(kf[(Q) & 1], Q, T, hi, s_next[Q][T]);                 \
    else                                                                          \
      s_next[Q][T] = DSX_QK(kf[(Q) & 1], Q, T, lo, zero4);                        \
  }
          DSX_STEP(0, 0) DSX_STEP(0, 1) DSX_STEP(1, 0) DSX_STEP(1, 1) DSX_STEP(2, 0) DSX_STEP(2, 1) DSX_STEP(3, 0) DSX_STEP(3, 1)
#undef DSX_STEP
          // (pinned: nothing in front of the next branch needs the products, and they would be sunk behind it, away from the
          // vector work that is to run beside them)
          if (high) asm volatile("" : "+v"(s_next[q][col]));
          if (x == 5) kf[0] = k_frag(st1, 2);
          if (x == 7) kf[1] = k_frag(st1, 3);
          if (x == 12) {
#pragma unroll
            for (int f = 0; f < kAhead; ++f) vf[f] = v_frag(buf, f);
          }
          // 32 - kExpEarly entries spread over 16 slots
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if ((n - kExpEarly) * 16 < (x + 1) * (32 - kExpEarly)) exp_entry(s_cur, off_cur, inv_cur, pw_cur, n++);
          if (x == 4) issue_k(st3);
          if (x == 6) cv_write(buf ^ 1, raw);
          if (x == 10) issue_v(st3);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (UNI) {
          // A lane's sum over its keys bounds each of its weights: as long as it fits fp16, so do they, and the scores' own
          // maximum is not needed.  Otherwise (rows that see their first token among them, their weights being inf) the
          // scores are still there: move the references and make the tile's weights again.
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(lsum[0] > kMostSum || lsum[1] > kMostSum) != 0, 0)) {
            const float ev[kGroups] = {(float)(127 - (int)(__float_as_uint(inv_cur[0]) >> 23))};
            float mx[2];
            scan(s_cur, ev, mx);
            move(mx, pw_cur, false);
            offsets(ev, off_cur);
            lsum[0] = lsum[1] = 0.f;
#pragma unroll
            for (int n3 = 0; n3 < 32; ++n3) exp_entry(s_cur, off_cur, inv_cur, pw_cur, n3);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          l_run[t] = UNI ? __builtin_fmaf(lsum[t], inv_cur[0], l_run[t]) : l_run[t] + lsum[t];
          lsum[t] = 0.f;
        }
        // ---- stage 2
        if (wave >= 4) __builtin_amdgcn_s_setprio(0);
        float ev[kGroups];
        scale_floats(vs, ev, inv_next);
        auto pv = [&](int f, int t) {
          if (t == 0 && f + kAhead < 16) vf[(f + kAhead) % (kAhead + 1)] = v_frag(buf, f + kAhead);
          const int ch = f >> 3, i2 = f & 7;
          const u32x4 w = {pw_cur[ch][t][0], pw_cur[ch][t][1], pw_cur[ch][t][2], pw_cur[ch][t][3]};
          o[i2][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[f % (kAhead + 1)], __builtin_bit_cast(f16x8, w), o[i2][t],
                                                            0, 0, 0);
        };
#pragma unroll
        for (int f = 0; f < kScanFrags; ++f)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            pv(f, t);
            __builtin_amdgcn_sched_barrier(0);
          }
        if (__builtin_expect(more, 1)) {
          mask(s_next, kb + 1);
          if constexpr (!UNI) {
            float mx[2];
            scan(s_next, ev, mx);
            if (__builtin_expect(must_move(mx), 0)) move(mx, pw_cur, true);
          }
        }
        offsets(ev, off_next);
        __builtin_amdgcn_sched_barrier(0);
        // (in the last interval the entries below come from a tile that does not exist; they and lsum are dropped)
        int n2 = 0;
#pragma unroll
        for (int f = kScanFrags; f < 16; ++f)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            pv(f, t);
            // for the next interval: scalar work, which at its head would have nothing beside it
            if (f == 5 && t == 0) scales_of(kb + 2, ks, vs);
            if (f == 9 && t == 0) aim(kb + 4);
            // kExpEarly entries spread over the slots that are left
            if (n2 * 2 * (16 - kScanFrags) < (2 * (f - kScanFrags) + t + 1) * kExpEarly)
              exp_entry(s_next, off_next, inv_next, pw_next, n2++);
            __builtin_amdgcn_sched_barrier(0);
          }
        if (__builtin_expect(boundary(kb), 0)) nan_rows(kb, buf, i & 3);
      }
    };

    aim(kb_begin);
    issue_k(0);
    issue_v(0);
    aim(kb_begin + 1);
    issue_k(1);
    issue_v(1);
    aim(kb_begin + 2);
    issue_k(2);
    issue_v(2);
    scales_of(kb_begin, ks, vs);
    DSX_HEAD(4);
    {
      uint32_t raw[4];
      cv_read(0, raw);
      if (boundary(kb_begin)) cv_fix(kb_begin, 0, raw);
      cv_write(0, raw);
      if (active) {
        i32x8 kf;
#define DSX_FIRST(Q)                                 \
  kf = k_frag(0, Q);                                 \
  sA[Q][0] = DSX_QK(kf, Q, 0, lo, zero4);            \
  sA[Q][1] = DSX_QK(kf, Q, 1, lo, zero4);            \
  sA[Q][0] = DSX_QK(kf, Q, 0, hi, sA[Q][0]);         \
  sA[Q][1] = DSX_QK(kf, Q, 1, hi, sA[Q][1]);
        DSX_FIRST(0) DSX_FIRST(1) DSX_FIRST(2) DSX_FIRST(3)
#undef DSX_FIRST
        float ev[kGroups], mx[2];
        scale_floats(vs, ev, invA);
        mask(sA, kb_begin);
        scan(sA, ev, mx);
        move(mx, pwA, false);
        offsets(ev, offA);
#pragma unroll
        for (int n = 0; n < kExpEarly; ++n) exp_entry(sA, offA, invA, pwA, n);
      }
    }
    if (!active) {  // a wave without rows: its loads and its share of the conversion
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const int i = kb - kb_begin;
        uint32_t raw[4];
        aim(kb + 3);
        DSX_HEAD(2);
        cv_read((i + 1) & 3, raw);
        issue_k((i + 3) & 3);
        issue_v((i + 3) & 3);
        if (boundary(kb + 1)) cv_fix(kb + 1, (i + 1) & 1, raw);
        cv_write((i + 1) & 1, raw);
      }
    }
    scales_of(kb_begin + 1, ks, vs);
    aim(kb_begin + 3);
    for (int kb = kb_begin; active && kb < kb_end; kb += 2) {
      interval(kb, 0, sA, sB, pwA, pwB, offA, invA, offB, invB);
      if (kb + 1 < kb_end) interval(kb + 1, 1, sB, sA, pwB, pwA, offB, invB, offA, invA);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the direct loads that nobody reads
#undef DSX_QK
#undef DSX_HEAD
  }
  if (!active) return;

#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float l = quad_sum(l_run[t]);
    const int r = wave * 32 + 16 * t + n16;  // row of the unit
    const int pr = pr0 + r;
    if (unit >= a.first_split) {
      const int64_t at = ((unit - a.first_split) * a.splits + split) * kTileRows + r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *reinterpret_cast<f32x4*>(a.part_o + at * kKvDim + 32 * g4 + 8 * e + i) =
              f32x4{o[i][t][e], o[i + 1][t][e], o[i + 2][t][e], o[i + 3][t][e]};
      if (g4 == 0) {
        a.part_ml[2 * at] = m_ref[t] == kNoRef ? -INFINITY : m_ref[t];
        a.part_ml[2 * at + 1] = l;
      }
    } else if (pr < packed) {
      const float inv = s.ok ? (l == 0.f ? 0.f : 1.f / l) : NAN;
      const int row = a.by_group(pr), hh = h * a.group + pr - row * a.group;
      uint16_t* dst = (uint16_t*)a.p.out + times(s.row0 + row, a.p.o_sr) + times(hh, a.p.o_sh) + 32 * g4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(o[2 * i][t][e] * inv, o[2 * i + 1][t][e] * inv);
        *reinterpret_cast<u32x4*>(dst + 8 * e) = w;
      }
    }
  }
}

}  // namespace

// The units behind the last full round of workgroups leave compute units idle: when at least two pieces of each fit
// into one round, and a piece is long enough to be worth its partial result (a join costs about as much as eight tiles),
// their key ranges are cut.
void kv_tile_split(int64_t units, int64_t span, int cus, int64_t& tail, int& pieces) {
  const int64_t tiles = (span + KB - 1) / KB;
  tail = units % cus;
  const int64_t fit = tail > 0 ? cus / tail : 1;
  const int64_t most = tiles / 8;
  pieces = (int)(fit < most ? fit : most);
  if (pieces > 64) pieces = 64;
  if (pieces < 2) {
    pieces = 1;
    tail = 0;
  }
}

int launch_kv_tile(const AttnArgs& a, int64_t units, hipStream_t st) {
  static PerDeviceOnce attr_once;
  const int attr_rc = per_device_once(attr_once, [](int) {
    for (const void* f : {(const void*)kv_tile_kernel<true>, (const void*)kv_tile_kernel<false>})
      if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes) != hipSuccess)
        return (int)DSX_ELAUNCH;
    return (int)DSX_OK;
  });
  if (attr_rc != DSX_OK) return attr_rc;
  const int64_t whole8 = (a.first_split + 7) & ~7ll, cut8 = ((units - a.first_split) * a.splits + 7) & ~7ll;
  const dim3 grid((unsigned)(whole8 + cut8)), block(512);
  if (a.c.page_size >= KB)
    kv_tile_kernel<true><<<grid, block, kLdsBytes, st>>>(a, units, (int)whole8, (int)cut8);
  else
    kv_tile_kernel<false><<<grid, block, kLdsBytes, st>>>(a, units, (int)whole8, (int)cut8);
  return DSX_OK;
}

}  // namespace dsx
