// What the paged 8-bit key/value cache's kernels share: the cache's addressing with its bounds, and the block scale.
// Everything here also compiles for the host (dsx_kv_plan_check walks the same functions).
#pragma once
#include "common.h"

namespace dsx {

constexpr int kKvDim = 128;
constexpr int kScaleMin = -48, kScaleMax = 48;  // exponents a block scale takes (why: kv_attn.hip)

// Division of numbers below 2^31 by a number that the host knows: n * m >> shift with m = ceil(2^shift / d) and
// shift = 31 + ceil(log2 d) is floor(n / d) for those, and two scalar instructions instead of some fifteen.  (A short
// call's kernels spent a quarter of their time dividing.)
struct Divisor {
  uint32_t m, shift;
  __host__ static Divisor of(uint32_t d) {
    uint32_t log = 0;
    while ((1ull << log) < d) ++log;
    return {(uint32_t)(((1ull << (31 + log)) + d - 1) / d), 31 + log};
  }
  __host__ __device__ uint32_t operator()(uint32_t n) const { return (uint32_t)((uint64_t)n * m >> shift); }
};

// Page and row strides and the table's are held below 2^31 by the host's checks: one multiplication 32 x 32 -> 64 bits.
__host__ __device__ inline int64_t times(int n, int64_t stride) { return (int64_t)((uint64_t)(uint32_t)n * (uint32_t)stride); }

// One sequence of a packed batch.  The lengths live on the device and nothing on the host has seen them, so every
// kernel checks them against the bounds the host has checked the buffers with: `ok` false means that nothing of the
// sequence may be touched but its output rows, and `rows` is 0 when not even those can be named.
struct KvSeq {
  int row0, rows, kv;
  bool ok;
};
__host__ __device__ inline KvSeq kv_seq(const dsx_kv_batch& n, int b, int64_t total_rows) {
  const int r0 = n.row_start[b], r1 = n.row_start[b + 1];
  int kv = n.kv_len[b];
#ifdef __HIP_DEVICE_COMPILE__
  asm volatile("" : "+v"(kv));  // (loaded along with the rows, not behind a look at them: a trip to memory less)
#endif
  if (r0 < 0 || r1 < r0 || r1 > total_rows) return {0, 0, 0, false};
  const bool ok = r1 - r0 <= n.max_rows && kv >= 0 && kv <= n.max_kv_len;
  return {r0, r1 - r0 <= n.max_rows ? r1 - r0 : n.max_rows, ok ? kv : 0, ok};
}

// Tokens [begin, end) that row i of a sequence sees.
__host__ __device__ inline void kv_row_span(int kv, int rows, int i, int causal, int window, int& begin, int& end) {
  end = causal ? kv - rows + i + 1 : kv;
  if (end < 0) end = 0;
  begin = window > 0 && end > window ? end - window : 0;
}

// Smallest e in [kScaleMin, kScaleMax] with amax <= 448 * 2^e (448 = 1.75 * 2^8); amax finite, >= 0.
__host__ __device__ inline int kv_block_exponent(uint32_t amax_bits) {
  int e = (int)(amax_bits >> 23) - 127 - 8;
  if ((amax_bits & 0x7fffffu) > 0x600000u) ++e;
  return e < kScaleMin ? kScaleMin : e > kScaleMax ? kScaleMax : e;
}

// Host checks of the part both calls share, and of packed rows.
bool kv_rows_ok(const void* p, int64_t sr, int64_t sh);
int kv_check_cache(const dsx_kv_cache* c, const dsx_kv_batch* n, int64_t total_rows);

}  // namespace dsx
