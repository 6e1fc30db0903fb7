// Tokens' positions and their places in a paged cache, and the turns of rotary
// positions: what the kernels that walk over new tokens' rows share.
#pragma once

#include "rkv_common.h"

namespace rkv {
namespace {

struct Places {
  const void* positions;     // int32 or int64 per token (null: from the sequences)
  int wide_positions;
  // paged: token t belongs to the sequence b with starts[b] <= t < starts[b + 1]
  // (null: sequence t), at position lengths[b] - (starts[b + 1] - t)
  const int32_t* starts;
  const int32_t* lengths;
  const int32_t* table;
  int64_t table_stride;
  int sequences, max_blocks, pages, shift;
};

// Where a token's rows go: its position, and its page and row in a cache
// (page < 0: not in the cache).
struct Place {
  int64_t position;
  int page, row;
  bool live;  // has a position: its rows turn
};

__device__ __forceinline__ Place place_of(const Places& a, int64_t t) {
  Place p{0, -1, 0, true};
  if (a.positions) {
    p.position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[t]
                                  : static_cast<const int32_t*>(a.positions)[t];
    return p;
  }
  int64_t b = t, behind = 1;  // tokens of the sequence from this one on
  if (a.starts) {
    // the first sequence that ends after t (empty ones end where they start)
    int lo = 0, hi = a.sequences;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid + 1] <= t) lo = mid + 1;
      else hi = mid;
    }
    b = lo;
    if (b >= a.sequences || a.starts[b] > t) return Place{0, -1, 0, false};
    behind = a.starts[b + 1] - t;
  }
  p.position = (int64_t)a.lengths[b] - behind;
  if (p.position < 0) return Place{0, -1, 0, false};
  const int64_t block = p.position >> a.shift;
  if (block < a.max_blocks) {
    const int page = a.table[b * a.table_stride + block];
    p.page = page >= 0 && page < a.pages ? page : -1;
  }
  p.row = (int)(p.position & ((1 << a.shift) - 1));
  return p;
}

// cos and sin of `quarters` quarter turns, to an ulp or two of fp32 (rms error
// 2.0e-8, at most 9.5e-8, and 1.9e-7 of a sine).  The
// angle of a far position needs more than fp32's 24 bits (131071 * 1 rad has
// an ulp of 0.008 rad there), so the whole quarters are taken off in fp64:
// adding 1.5 * 2^52 leaves them in the sum's low bits, rounded to nearest.
// What is left, at most pi/4, is rounded twice (once, with the product in fp64,
// would leave 1.5e-8 of the sine's rms) and goes through the Taylor series of sin (to a^9,
// truncation 2e-9) and cos (to a^10, 2e-10).
__device__ __forceinline__ void cos_sin(double quarters, float& c, float& s) {
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
  const double sum = quarters + kWhole;
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, sum);
  const float a = (float)(quarters - (sum - kWhole)) * 1.57079632679489662f;
  const float a2 = a * a;
  float p = 2.75573192239858907e-06f;                    // 1/9!
  p = __builtin_fmaf(p, a2, -1.98412698412698413e-04f);  // 1/7!
  p = __builtin_fmaf(p, a2, 8.33333333333333333e-03f);   // 1/5!
  p = __builtin_fmaf(p, a2, -1.66666666666666667e-01f);  // 1/3!
  const float sn = __builtin_fmaf(p * a2, a, a);
  float q = -2.75573192239858907e-07f;                   // 1/10!
  q = __builtin_fmaf(q, a2, 2.48015873015873016e-05f);   // 1/8!
  q = __builtin_fmaf(q, a2, -1.38888888888888889e-03f);  // 1/6!
  q = __builtin_fmaf(q, a2, 4.16666666666666667e-02f);   // 1/4!
  q = __builtin_fmaf(q, a2, -0.5f);
  const float cn = __builtin_fmaf(q, a2, 1.0f);
  // quarter 0 (c, s), 1 (-s, c), 2 (-c, -s), 3 (s, -c)
  const bool swap = (k & 1u) != 0u;
  c = bits_f32(f32_bits(swap ? sn : cn) ^ ((k + 1u) << 30 & 0x80000000u));
  s = bits_f32(f32_bits(swap ? cn : sn) ^ (k << 30 & 0x80000000u));
}

}  // namespace
}  // namespace rkv
