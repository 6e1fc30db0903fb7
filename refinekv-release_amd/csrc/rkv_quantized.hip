// A paged KV cache in 4 bits: the append of new tokens' keys and values
// (rkv_quantized_append), the rows that its tokens stand for
// (rkv_quantized_read) and the attention of one new token per sequence over it
// (rkv_quantized_decode).
//
// Every 32 dims of a row are a group with a scale s and a zero z, both fp16:
//   z = min, s = (max - min) / 15, code = round((x - z) / s) in 0..15,
// and stand for z + s code.  s is rounded up to 7 significant bits, so that
// s code is an fp16 number: the matrix products take it as it is, and the
// zeros' share of a sum comes from a product of its own, so that nothing is
// rounded between the codes and the fp32 sums.  A group with a value that is
// not finite, or past 4096 in magnitude, has NaN for both.
//
// A row of d dims is d / 2 bytes of codes and d / 8 of scales: 160 bytes a token
// of keys and values at d 128, where 16 bits take 512.  Both lie as the decode's
// lanes load them, in whole vectors:
//   keys' codes   [token][lane row lg of 4][group]: a dword of dims 32 group +
//                 8 lg .. + 7, dim 2 i at bit 4 i, 2 i + 1 at 4 i + 16.
//   keys' scales  [token][group]: s, z.
//   values' codes [4 tokens][piece][column i of 16]: E = 8, 4 or 2 dims from
//                 E i of a piece of 128, 64 or 32 dims, E / 2 dwords; in the
//                 list of (token pair, dim) entry m lies in dword m / 4 at bit
//                 4 (m % 4), the pair's second token 16 bits on.
//   values' scales [4 tokens][group]: s of the tokens 0 .. 3, z of them.
#include "rkv_paged_walk.h"
#include "rkv_places.h"

namespace rkv {
namespace {

// In magnitude, of a group's values: 64 times a scale (at most 8192 / 15, and 1/64
// more) stays in fp16's range.
constexpr float kLargest = 4096.0f;
constexpr int kGroupDims = 32;

typedef _Float16 Half2 __attribute__((ext_vector_type(2)));
typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef uint32_t U32x3 __attribute__((ext_vector_type(3)));

__device__ __forceinline__ Half2 half2_of(uint32_t w) { return __builtin_bit_cast(Half2, w); }
__device__ __forceinline__ uint32_t word_of(Half2 h) { return __builtin_bit_cast(uint32_t, h); }

// ---------------------------------------------------------------------------
// Append and read
// ---------------------------------------------------------------------------

constexpr int kRowThreads = 256;
constexpr int kItem = 8;  // dims of a thread: 16 bytes of a row
// From so many threads on the device is full, and fewer threads turn more heads
// each with the same cos and sin.
constexpr int64_t kManyRowThreads = 4 * 1024 * 64;

template <typename T>
using Item = T __attribute__((ext_vector_type(kItem)));

struct Pool {
  char* codes;
  char* scales;
};

struct QuantRows : Places {
  const char* src[3];               // queries, keys, values (heads 0: absent)
  char* dst[3];                     // turned queries; (read) keys, values
  int64_t src_ts[3], src_hs[3];     // token and head strides, elements
  int64_t dst_ts, dst_hs;           // of the turned queries
  int q_heads, heads;               // query heads, KV heads
  int64_t tokens;
  int dim, rotary_dim, interleaved;
  const double* rates;
  float scale;                      // attention factor
  Pool keys, values;
  int slots, per_block;             // heads a token's threads hold at a time, a workgroup's tokens
};

// The row's place in a pool, in rows of a page's head.
__device__ __forceinline__ int64_t row_at(const QuantRows& a, const Place& p, int h) {
  return (((int64_t)p.page * a.heads + h) << a.shift) + p.row;
}

// Where a value row's codes of dims d0 .. d0 + 7 lie in its 4 tokens' block, as
// the bytes of column `i`, `E` dims of one token each.
struct ValuePiece {
  int base, dims;  // the piece's byte in the block, dims of a column
  int column;      // the item's first column
};

__device__ __forceinline__ ValuePiece value_piece(int dim, int d0) {
  const int whole = dim & ~127;
  if (d0 < whole) return ValuePiece{(d0 & ~127) * 2, 8, (d0 & 127) / 8};
  const int half = dim & 64;
  if (half && d0 < whole + 64) return ValuePiece{whole * 2, 4, (d0 - whole) / 4};
  return ValuePiece{(whole + half) * 2, 2, (d0 - whole - half) / 2};
}

// The largest value and (min of the negatives) the smallest over a quad's
// lanes, the 4 items of a group.
template <int kCtrl>
__device__ __forceinline__ float quad_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl,
                                                               0xF, 0xF, false));
}
__device__ __forceinline__ float quad_max(float v) {
  v = __builtin_fmaxf(v, quad_lane<0xB1>(v));
  return __builtin_fmaxf(v, quad_lane<0x4E>(v));
}

// A group's scale and zero from its lanes' values, and the item's codes as whole
// floats.
template <typename T>
__device__ __forceinline__ void quantize(const Item<T>& v, uint32_t& scale_zero,
                                         float (&code)[kItem]) {
  float x[kItem];
#pragma unroll
  for (int e = 0; e < kItem; ++e) x[e] = (float)v[e];
  float low = x[0], high = x[0];
#pragma unroll
  for (int e = 1; e < kItem; ++e) {
    low = __builtin_fminf(low, x[e]);
    high = __builtin_fmaxf(high, x[e]);
  }
  // the largest magnitude as an integer: NaN's are the largest of all (min and
  // max would skip them)
  typedef uint16_t U16x2 __attribute__((ext_vector_type(2)));
  const U32x4 words = __builtin_bit_cast(U32x4, v);
  U16x2 size = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    size = __builtin_elementwise_max(size, __builtin_bit_cast(U16x2, words[i] & 0x7fff7fffu));
  uint32_t top = size[0] > size[1] ? size[0] : size[1];
  constexpr uint32_t kTop = __builtin_bit_cast(uint16_t, (T)kLargest);
  const float over = top > kTop ? 1.0f : 0.0f;
  high = quad_max(high);
  low = -quad_max(-low);
  const bool held = quad_max(over) == 0.0f;
  const _Float16 near = (_Float16)((high - low) / 15.0f), zero = (_Float16)low;
  const uint32_t up = ((uint32_t)__builtin_bit_cast(uint16_t, near) + 15u) & 0xfff0u;
  const float step = (float)__builtin_bit_cast(_Float16, (uint16_t)up), base = (float)zero;
  scale_zero = held ? up | (uint32_t)__builtin_bit_cast(uint16_t, zero) << 16 : 0x7e007e00u;
  // (x - zero) / scale, correctly rounded: with the reciprocal so, a quotient's
  // remainder corrects it (Markstein).  A reciprocal of 0 where there is no
  // scale gives codes of 0 (and NaN, which the maximum makes 0).
  const float per = held && step > 0.0f ? 1.0f / step : 0.0f;
#pragma unroll
  for (int e = 0; e < kItem; ++e) {
    const float d = x[e] - base, near_q = d * per;
    const float q = __builtin_fmaf(__builtin_fmaf(-near_q, step, d), per, near_q);
    code[e] = __builtin_rintf(__builtin_fminf(__builtin_fmaxf(q, 0.0f), 15.0f));
  }
}

// Four codes, 4 bits each, low first.
__device__ __forceinline__ uint32_t pack(float c0, float c1, float c2, float c3) {
  return (uint32_t)__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c3, 16.0f, c2), 16.0f, c1), 16.0f,
                                  c0);
}

__device__ __forceinline__ void store_key(const QuantRows& a, int64_t row, int d0,
                                          uint32_t scale_zero, const float (&code)[kItem]) {
  const int groups = a.dim / kGroupDims, group = d0 / kGroupDims, lg = d0 % kGroupDims / kItem;
  const uint32_t w = pack(code[0], code[2], code[4], code[6]) |
                     pack(code[1], code[3], code[5], code[7]) << 16;
  reinterpret_cast<uint32_t*>(a.keys.codes + row * (a.dim / 2))[lg * groups + group] = w;
  if (lg == 0) reinterpret_cast<uint32_t*>(a.keys.scales)[row * groups + group] = scale_zero;
}

__device__ __forceinline__ void store_value(const QuantRows& a, int64_t row, int d0,
                                            uint32_t scale_zero, const float (&code)[kItem]) {
  const int token = (int)(row & 3), pair = token / 2, second = token % 2;
  const ValuePiece at = value_piece(a.dim, d0);
  char* block = a.values.codes + (row >> 2) * (2 * a.dim) + at.base;
  const uint32_t low = pack(code[0], code[1], code[2], code[3]),
                 high = pack(code[4], code[5], code[6], code[7]);
  if (at.dims > 2) {
    // (8 dims: two words of a column; 4: one each of two columns)
    char* to = block + (at.dims == 8 ? at.column * 16 + pair * 8 : at.column * 8 + pair * 4) +
               second * 2;
    *reinterpret_cast<uint16_t*>(to) = (uint16_t)low;
    *reinterpret_cast<uint16_t*>(to + (at.dims == 8 ? 4 : 8)) = (uint16_t)high;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<uint8_t*>(block + (at.column + k) * 4 + second * 2 + pair) =
          (uint8_t)((k < 2 ? low : high) >> (8 * (k % 2)));
  }
  if (d0 % kGroupDims == 0) {
    char* s = a.values.scales + (row >> 2) * (a.dim / 2) + d0 / kGroupDims * 16 + token * 2;
    *reinterpret_cast<uint16_t*>(s) = (uint16_t)scale_zero;
    *reinterpret_cast<uint16_t*>(s + 8) = (uint16_t)(scale_zero >> 16);
  }
}

// Where an item's partners in a turn are, the dims rotary_dim / 2 away or
// (interleaved) the neighbours: in the item itself, in an item of their own, in
// parts of two; or (the whole head turns) in the thread's second item.
enum Partner : int { kWithin, kWhole, kParts, kHalves };

// Memory and vector issue bound it together: 18 K tokens' rows of 28 + 4 + 4 heads
// (d 128, fp16, 150 MB in and out) in 33 us, 4.5 TB/s, of which some 23 us are
// vector instructions (a cos and sin costs 30, a coded value 8).  Coding in the
// same pass as the queries 42 us, with a division a value 50, each half of a row
// in a thread of its own (which works out the other's cos and sin again) 77.
// A thread holds 8 dims of a token's rows (kHalves: twice 8, half a row apart):
// it works out their cos and sin once and applies them to every slots-th head,
// queries, then keys, then values, the next head's row on its way while one is
// turned; the 4 lanes of a group meet for its bounds.
template <typename T, int kPartner>
__global__ __launch_bounds__(kRowThreads) void quantize_rows_kernel(QuantRows a) {
  using V = Item<T>;
  constexpr int kVecs = kPartner == kHalves ? 2 : 1;
  const int items = a.dim / (kItem * kVecs), wide = items * a.slots;
  const int in_block = (int)threadIdx.x / wide, rest = (int)threadIdx.x % wide;
  const int slot = rest / items, d0 = rest % items * kItem;
  const int64_t t = (int64_t)blockIdx.x * a.per_block + in_block;
  if (in_block >= a.per_block || t >= a.tokens) return;
  const int half = a.rotary_dim / 2;
  const bool in_part = d0 < a.rotary_dim;
  // the second load: the partners' (kWhole), or the second item
  const int from = kPartner == kHalves ? d0 + half
                   : !in_part          ? d0
                   : d0 < half         ? d0 + half
                                       : d0 - half;
  V v, w;
  const T* row;
  auto load = [&]() {
    v = *reinterpret_cast<const V*>(row + d0);
    if constexpr (kPartner == kWhole || kPartner == kHalves)
      w = *reinterpret_cast<const V*>(row + from);
  };
  // (the thread's heads: every slots-th of the queries, then of keys and values)
  auto to_key_value = [&](int n) {
    const bool value = n >= a.heads;
    row = reinterpret_cast<const T*>(value ? a.src[2] : a.src[1]) +
          t * (value ? a.src_ts[2] : a.src_ts[1]) +
          (value ? n - a.heads : n) * (value ? a.src_hs[2] : a.src_hs[1]);
  };
  if (slot < a.q_heads)
    row = reinterpret_cast<const T*>(a.src[0]) + t * a.src_ts[0] + slot * a.src_hs[0];
  else
    to_key_value(min(slot, 2 * a.heads - 1));
  load();
  const Place place = place_of(a, t);
  const bool turns = place.live && in_part;
  float c[kItem], s[kItem];  // (s with the sign that the item's dims take it with)
  if (turns) {
    const double position4 = 4.0 * (double)place.position;  // rates are whole turns
    constexpr int kPairs = kPartner == kWithin ? kItem / 2 : kItem;
    double rate[kPairs];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      // (dims of the last item that pass have no pair)
      const int d = kPartner == kWithin ? d0 / 2 + e : d0 + e < half ? d0 + e : d0 + e - half;
      rate[e] = a.rates[min(d, half - 1)];
    }
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      float cs, sn;
      cos_sin(position4 * rate[e], cs, sn);
      cs *= a.scale;
      sn *= a.scale;
      if constexpr (kPartner == kWithin) {
        c[2 * e] = c[2 * e + 1] = cs;
        s[2 * e] = -sn;
        s[2 * e + 1] = sn;
      } else {
        c[e] = cs;
        s[e] = d0 + e < half ? -sn : sn;
      }
    }
  }
  auto turn = [&](V& x, V& y, const T* from_row) {
    const V x0 = x, y0 = y;
#pragma unroll
    for (int e = 0; e < kItem; ++e) {
      const int d = d0 + e;
      if constexpr (kPartner == kHalves) {
        x[e] = (T)__builtin_fmaf((float)x0[e], c[e], (float)y0[e] * s[e]);
        y[e] = (T)__builtin_fmaf((float)y0[e], c[e], -((float)x0[e] * s[e]));
      } else {
        float other;
        if constexpr (kPartner == kWithin) other = (float)x0[e ^ 1];
        else if constexpr (kPartner == kWhole) other = (float)y0[e];
        else other = d < a.rotary_dim ? (float)from_row[d < half ? d + half : d - half] : 0.0f;
        if (d < a.rotary_dim) x[e] = (T)__builtin_fmaf((float)x0[e], c[e], other * s[e]);
      }
    }
  };
  if (a.q_heads > 0) {
    T* to = reinterpret_cast<T*>(a.dst[0]) + t * a.dst_ts + slot * a.dst_hs;
    for (int n = slot; n < a.q_heads; n += a.slots) {
      V x = v, y = w;
      const T* const from_row = row;
      if (n + a.slots < a.q_heads) row += a.slots * a.src_hs[0];
      else to_key_value(min(slot, 2 * a.heads - 1));
      load();
      if (turns) turn(x, y, from_row);
      *reinterpret_cast<V*>(to + d0) = x;
      if constexpr (kPartner == kHalves) *reinterpret_cast<V*>(to + from) = y;
      to += a.slots * a.dst_hs;
    }
  }
  if (place.page < 0) return;
  // (keys and values after the queries: the wave's lanes code together)
  for (int n = slot; n < 2 * a.heads;) {
    V x = v, y = w;
    const T* const from_row = row;
    const int here = n;
    n += a.slots;
    if (n < 2 * a.heads) {
      to_key_value(n);
      load();
    }
    const bool key = here < a.heads;
    if (key && turns) turn(x, y, from_row);
    const int64_t at = row_at(a, place, key ? here : here - a.heads);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      uint32_t scale_zero;
      float code[kItem];
      quantize<T>(k ? y : x, scale_zero, code);
      if (key) store_key(a, at, k ? from : d0, scale_zero, code);
      else store_value(a, at, k ? from : d0, scale_zero, code);
    }
  }
}

// The rows that tokens of the cache stand for, in the cache's type: zeros for a
// token without a position, NaN for one whose page is not the cache's.
template <typename T>
__global__ __launch_bounds__(kRowThreads) void quantized_read_kernel(QuantRows a) {
  typedef T V __attribute__((ext_vector_type(kItem)));
  const int items = a.dim / kItem, wide = items * a.slots;
  const int in_block = (int)threadIdx.x / wide, rest = (int)threadIdx.x % wide;
  const int slot = rest / items, d0 = rest % items * kItem;
  const int64_t t = (int64_t)blockIdx.x * a.per_block + in_block;
  if (in_block >= a.per_block || t >= a.tokens) return;
  const Place place = place_of(a, t);
  const int groups = a.dim / kGroupDims, group = d0 / kGroupDims;
  for (int n = slot; n < 2 * a.heads; n += a.slots) {
    const bool key = n < a.heads;
    const int h = key ? n : n - a.heads;
    V v;
    if (place.page < 0) {
      const float fill = place.live ? __builtin_nanf("") : 0.0f;
#pragma unroll
      for (int e = 0; e < kItem; ++e) v[e] = (T)fill;
    } else {
      const int64_t row = row_at(a, place, h);
      uint32_t code[kItem];
      float step, zero;
      if (key) {
        const int lg = d0 % kGroupDims / kItem;
        const uint32_t w = reinterpret_cast<const uint32_t*>(
            a.keys.codes + row * (a.dim / 2))[lg * groups + group];
        const Half2 sz =
            half2_of(reinterpret_cast<const uint32_t*>(a.keys.scales)[row * groups + group]);
        step = (float)sz[0];
        zero = (float)sz[1];
#pragma unroll
        for (int e = 0; e < kItem; ++e) code[e] = w >> (4 * (e / 2) + 16 * (e % 2)) & 15u;
      } else {
        const int token = (int)(row & 3), pair = token / 2, second = token % 2;
        const ValuePiece at = value_piece(a.dim, d0);
        const char* block = a.values.codes + (row >> 2) * (2 * a.dim) + at.base;
#pragma unroll
        for (int e = 0; e < kItem; ++e) {
          // (column, entry of the list) of the dim
          const int column = at.column + e / at.dims, m = pair * at.dims + e % at.dims;
          const uint32_t w = *reinterpret_cast<const uint16_t*>(
              block + (column * (at.dims / 2) + m / 4) * 4 + second * 2);
          code[e] = w >> (4 * (m % 4)) & 15u;
        }
        const char* sz = a.values.scales + (row >> 2) * (a.dim / 2) + group * 16 + token * 2;
        step = (float)*reinterpret_cast<const _Float16*>(sz);
        zero = (float)*reinterpret_cast<const _Float16*>(sz + 8);
      }
#pragma unroll
      for (int e = 0; e < kItem; ++e) v[e] = (T)__builtin_fmaf((float)code[e], step, zero);
    }
    T* to = reinterpret_cast<T*>(a.dst[key ? 1 : 2]) + (t * a.heads + h) * a.dim + d0;
    *reinterpret_cast<V*>(to) = v;
  }
}

// ---------------------------------------------------------------------------
// Decode
// ---------------------------------------------------------------------------

struct QuantArgs : WalkArgs {
  const char* key_codes;
  const char* key_scales;
  const char* value_codes;
  const char* value_scales;
};

// Cache policy of the loads of codes and scales: non-temporal, as a token is
// read once a step (8 x 131072 tokens 258 -> 254 us, 64 ragged ones 57.2 -> 55.9).
constexpr int kStreamCodes = 2;

// N dwords from consecutive places of a view.
template <int N>
__device__ __forceinline__ void load_words(__amdgpu_buffer_rsrc_t view, uint32_t at,
                                           uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i + 4 <= N; i += 4) {
    const U32x4 v = __builtin_amdgcn_raw_buffer_load_b128(view, (int)(at + 4u * i), 0, kStreamCodes);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i + j] = v[j];
  }
  constexpr int kDone = N / 4 * 4;
  if constexpr (N % 4 == 3) {
    const U32x3 v = __builtin_amdgcn_raw_buffer_load_b96(view, (int)(at + 4u * kDone), 0, kStreamCodes);
#pragma unroll
    for (int j = 0; j < 3; ++j) w[kDone + j] = v[j];
  } else if constexpr (N % 4 == 2) {
    const U32x2 v = __builtin_amdgcn_raw_buffer_load_b64(view, (int)(at + 4u * kDone), 0, kStreamCodes);
    w[kDone] = v[0];
    w[kDone + 1] = v[1];
  } else if constexpr (N % 4 == 1) {
    w[kDone] = __builtin_amdgcn_raw_buffer_load_b32(view, (int)(at + 4u * kDone), 0, kStreamCodes);
  }
}

// Entry m of 4 that a word holds: the two codes as fp16 numbers 64 + code (the
// code in bits 4 .. 7 of 64, whose last bit is 1/16).
// Mask and 64 come in registers: as literals they take an instruction each.
struct CodeBits {
  uint32_t mask = 0x00f000f0u, sixty_four = 0x54005400u;
  __device__ __forceinline__ CodeBits() {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(sixty_four));
  }
};

template <int M>
__device__ __forceinline__ Half2 codes_of(const CodeBits& bits, uint32_t w) {
  const uint32_t at = M == 0 ? w << 4 : w >> (4 * M - 4);
  return half2_of((at & bits.mask) | bits.sixty_four);
}

// The walk's operands from 4-bit pages.  All products run on fp16: a code times
// its scale is (64 + code) s - 64 s, one fused operation without a rounding (7
// bits times 7).  A query row enters scaled by a power of two that makes its
// largest value 1 to 2, so that bf16 ones fit (what falls below fp16's range is
// 2^-24 of the largest at most); the sums of its values over the groups, which
// the keys' zeros are multiplied with, enter in three parts that hold fp32's 24
// bits.
template <int D, bool kHalf_, bool kScores>
struct Pages4 {
  static constexpr int kDim = D;
  // (kRareEnds: a row's last tile is a branch, not selects in every tile)
  static constexpr bool kHalf = kHalf_, kScaleLate = true, kRareEnds = true;
  using Args = QuantArgs;
  using P = Pieces<D>;
  static constexpr int G = D / kGroupDims;
  static constexpr int kPieces = P::k8 + P::k4 + P::k2;
  static constexpr int kAccs = P::kBlocks + kPieces;  // the last: the zeros' share

  struct Tile {
    uint32_t kc[2][G], ks[2][G];        // keys' codes and scales of a half
    uint32_t vc[2][G];                  // values' codes
    U32x4 vs[2][kPieces];               // values' scales of 4 tokens, their zeros
  };
  struct Query {
    Half8 q[G];
    Half8 sums;   // lane row lg: part lg of the groups' sums
    float back;   // the power of two that was taken off
  };

  const Args& a;
  const int li, lg;
  const CodeBits bits;
  __device__ __forceinline__ Pages4(const Args& args, int li_, int lg_)
      : a(args), li(li_), lg(lg_) {}

  __device__ __forceinline__ void take(Query& q, const U32x4 (&rows)[G]) const {
    float x[G][8];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t w = rows[j][e / 2];
        if constexpr (kHalf) x[j][e] = (float)half2_of(w)[e % 2];
        else x[j][e] = bits_f32(e % 2 ? w & 0xffff0000u : w << 16);
        top = __builtin_fmaxf(top, __builtin_fabsf(x[j][e]));
      }
    float u, v;
    xor16_pair(top, u, v);
    top = __builtin_fmaxf(u, v);
    xor32_pair(top, u, v);
    top = __builtin_fmaxf(u, v);
    uint32_t e2 = f32_bits(top) >> 23;
    e2 = e2 < 1u ? 1u : e2 > 253u ? 253u : e2;
    float by = bits_f32((254u - e2) << 23);  // 2^(127 - e2)
    // (scores that are scaled late are scaled by a magnitude)
    if constexpr (!kScores) by = a.scale < 0.0f ? -by : by;
    q.back = bits_f32(e2 << 23);
    q.sums = Half8{};
#pragma unroll
    for (int j = 0; j < G; ++j) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 h = (_Float16)(x[j][e] * by);
        q.q[j][e] = h;
        sum += (float)h;
      }
      xor16_pair(sum, u, v);
      sum = u + v;
      xor32_pair(sum, u, v);
      sum = u + v;
      const _Float16 high = (_Float16)sum;
      const _Float16 mid = (_Float16)(sum - (float)high);
      const _Float16 low = (_Float16)(sum - (float)high - (float)mid);
      q.sums[j] = lg == 0 ? high : lg == 1 ? mid : lg == 2 ? low : (_Float16)0.0f;
    }
  }
  __device__ __forceinline__ float unit(const Query& q) const {
    return !kScores && a.scale < 0.0f ? -q.back : q.back;
  }

  // A row's zeros' share joins its accumulators.
  static __device__ __forceinline__ void finish(F32x4 (&acc)[kAccs]) {
#pragma unroll
    for (int n = 0; n < P::kBlocks; ++n) {
      const int piece = n < 8 * P::k8 ? n / 8 : n < 8 * P::k8 + 4 * P::k4 ? P::k8 : P::k8 + P::k4;
      acc[n] += acc[P::kBlocks + piece];
    }
  }

  // The loads of a tile, always as many (a tile or half that is not there
  // reads through an empty view).
  __device__ __forceinline__ bool load(const Cursor& c, Tile& t, bool there) const {
    bool bad = c.bad;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = c.tile * kTileTokens + 16 * s;
      const int rows = there ? min(c.length - at, 16) : 0;
      int page = s ? c.page1 : c.page0;
      const bool out = (uint32_t)page >= (uint32_t)a.pages;
      // (the pages of tokens that no query sees any more may be gone)
      bad |= out && rows > 0 && (!kScores || at + 15 >= c.length - a.window);
      page = out ? 0 : page;
      const bool any = rows > 0 && !out;
      const uint32_t in_page = any ? (uint32_t)at & ((1u << a.shift) - 1u) : 0u;
      const int64_t row = (((int64_t)page * a.heads + c.h) << a.shift) + in_page;
      const uint32_t n = any ? (uint32_t)rows : 0u, blocks = (n + 3u) / 4u;
      const auto kc = view_of(a.key_codes + row * (D / 2), n * (D / 2));
      const auto ks = view_of(a.key_scales + row * (4 * G), n * (4 * G));
      const auto vc = view_of(a.value_codes + row * (D / 2), blocks * (2 * D));
      const auto vs = view_of(a.value_scales + row * (4 * G), blocks * (16 * G));
      load_words(kc, (uint32_t)(li * (D / 2) + lg * (4 * G)), t.kc[s]);
      load_words(ks, (uint32_t)(li * (4 * G)), t.ks[s]);
      const uint32_t block = (uint32_t)lg * (2 * D);
#pragma unroll
      for (int c8 = 0; c8 < P::k8; ++c8) {
        uint32_t w[4];
        load_words(vc, block + 256u * c8 + 16u * li, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.vc[s][4 * c8 + i] = w[i];
        t.vs[s][c8] = __builtin_amdgcn_raw_buffer_load_b128(
            vs, (int)((uint32_t)lg * (16 * G) + 16u * (4 * c8 + li / 4)), 0, 0);
      }
      if constexpr (P::k4 > 0) {
        uint32_t w[2];
        load_words(vc, block + 256u * P::k8 + 8u * li, w);
        t.vc[s][4 * P::k8] = w[0];
        t.vc[s][4 * P::k8 + 1] = w[1];
        t.vs[s][P::k8] = __builtin_amdgcn_raw_buffer_load_b128(
            vs, (int)((uint32_t)lg * (16 * G) + 16u * (4 * P::k8 + li / 8)), 0, 0);
      }
      if constexpr (P::k2 > 0) {
        uint32_t w[1];
        load_words(vc, block + 256u * P::k8 + 128u * P::k4 + 4u * li, w);
        t.vc[s][G - 1] = w[0];
        t.vs[s][kPieces - 1] = __builtin_amdgcn_raw_buffer_load_b128(
            vs, (int)((uint32_t)lg * (16 * G) + 16u * (G - 1)), 0, 0);
      }
    }
    return bad;
  }

  static __device__ __forceinline__ F32x4 mma(const U32x4& x, Half8 y, F32x4 z) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Half8, x), y, z, 0, 0, 0);
  }

  __device__ __forceinline__ void scores(const Query& q, const Tile& t, float (&x)[8]) const {
    const Half2 down = {(_Float16)-64.0f, (_Float16)-64.0f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      F32x4 s4 = {0.0f, 0.0f, 0.0f, 0.0f};
      U32x4 zeros = {0u, 0u, 0u, 0u};  // the token's, 8 slots
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const uint32_t sz = t.ks[s][j], w = t.kc[s][j];
        const Half2 step = half2_of(__builtin_amdgcn_perm(sz, sz, 0x01000100u));
        const Half2 base = step * down;
        const U32x4 k = {word_of(__builtin_elementwise_fma(codes_of<0>(bits, w), step, base)),
                         word_of(__builtin_elementwise_fma(codes_of<1>(bits, w), step, base)),
                         word_of(__builtin_elementwise_fma(codes_of<2>(bits, w), step, base)),
                         word_of(__builtin_elementwise_fma(codes_of<3>(bits, w), step, base))};
        s4 = mma(k, q.q[j], s4);
        zeros[j / 2] |= j % 2 ? sz & 0xffff0000u : sz >> 16;
      }
      s4 = mma(zeros, q.sums, s4);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[4 * s + r] = s4[r];
    }
  }

  // (tokens from .. behind - 1 of the tile are seen)
  __device__ __forceinline__ void products(F32x4 (&acc)[kAccs], Tile& t, const float (&p)[8],
                                           int from, int behind) const {
    Half8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // one fp16 part of a weight holds it to 2^-12, an eighth of what a bf16
      // output is rounded by; for fp16 outputs a second one holds the rest
      hi[e] = (_Float16)p[e];
      if constexpr (kHalf) lo[e] = (_Float16)(p[e] - (float)hi[e]);
    }
    if (behind < kTileTokens || (kScores && from > 0)) {
      // hidden tokens' scales may be anything, NaN as well: zeros here
      asm volatile("");
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          const int token = 16 * s + 4 * lg + 2 * pair;
          const uint32_t seen = (token >= from && token < behind ? 0xffffu : 0u) |
                                (token + 1 >= from && token + 1 < behind ? 0xffff0000u : 0u);
#pragma unroll
          for (int k = 0; k < kPieces; ++k) {
            t.vs[s][k][pair] &= seen;
            t.vs[s][k][2 + pair] &= seen;
          }
        }
    }
    const Half2 down = {(_Float16)-64.0f, (_Float16)-64.0f};
    auto add = [&](int n, const U32x4& words) {
      acc[n] = mma(words, hi, acc[n]);
      if constexpr (kHalf) acc[n] = mma(words, lo, acc[n]);
    };
    auto piece = [&](int k, int n0, int w0, auto dims) {
      constexpr int E = dims();
      Half2 step[4], base[4];
      U32x4 zeros;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          step[2 * s + pair] = half2_of(t.vs[s][k][pair]);
          base[2 * s + pair] = step[2 * s + pair] * down;
          zeros[2 * s + pair] = t.vs[s][k][2 + pair];
        }
      add(P::kBlocks + k, zeros);
      auto product = [&](auto dim) {
        constexpr int n = dim();
        U32x4 words;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          constexpr int m0 = n, m1 = E + n;
          words[2 * s] = word_of(__builtin_elementwise_fma(codes_of<m0 % 4>(bits, t.vc[s][w0 + m0 / 4]),
                                                           step[2 * s], base[2 * s]));
          words[2 * s + 1] = word_of(__builtin_elementwise_fma(
              codes_of<m1 % 4>(bits, t.vc[s][w0 + m1 / 4]), step[2 * s + 1], base[2 * s + 1]));
        }
        add(n0 + n, words);
      };
      product(std::integral_constant<int, 0>());
      product(std::integral_constant<int, 1>());
      if constexpr (E >= 4) {
        product(std::integral_constant<int, 2>());
        product(std::integral_constant<int, 3>());
      }
      if constexpr (E == 8) {
        product(std::integral_constant<int, 4>());
        product(std::integral_constant<int, 5>());
        product(std::integral_constant<int, 6>());
        product(std::integral_constant<int, 7>());
      }
    };
#pragma unroll
    for (int c8 = 0; c8 < P::k8; ++c8) piece(c8, 8 * c8, 4 * c8, std::integral_constant<int, 8>());
    if constexpr (P::k4 > 0)
      piece(P::k8, 8 * P::k8, 4 * P::k8, std::integral_constant<int, 4>());
    if constexpr (P::k2 > 0)
      piece(kPieces - 1, P::kBlocks - 2, G - 1, std::integral_constant<int, 2>());
  }
};

// Workgroups per CU that share the tiles (as kPerCu): from two to three at head_dim
// 64, 48 sequences of up to 16000 tokens, 64.2 -> 55.5 us; 96, 40 of them, 31.0
// -> 36.7; 128, 64 ragged ones 53.6 -> 60.4; from one to two at 256, 24 of up to
// 12000, 45.6 -> 54.0.
template <int D>
constexpr int kPerCu4 = D <= 64 ? 3 : D <= 128 ? 2 : 1;

// HBM and vector issue bound it together: 1.34 GB of 8 x 131072 tokens (8 KV heads,
// group 4, d 128) in 222-264 us, 5.1-6.0 TB/s; 313 vector instructions a tile of 32
// tokens (176 of them turn its 8192 codes into fp16) keep the ALUs busy for 138 us
// of it.  (378 when masks and biases were literals and every tile had the selects
// of a row's end, and 258 us.)  A call of few tokens is paged_kernel's chain of
// latencies: one sequence of 2003 tokens 7.7 us, then 4.5 for the join.
template <int D, bool kHalf, bool kScores>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(kPerCu4<D>))) void quantized_kernel(QuantArgs a) {
  walk<Pages4<D, kHalf, kScores>, kScores>(a);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Span {
  const void* at;
  int64_t bytes;
};

bool spans_meet(Span a, Span b) {
  const uint64_t x = reinterpret_cast<uint64_t>(a.at), y = reinterpret_cast<uint64_t>(b.at);
  return a.bytes > 0 && b.bytes > 0 && x < y + (uint64_t)b.bytes && y < x + (uint64_t)a.bytes;
}

// (codes of keys and values, scales of keys and values)
void pool_spans(const rkv_quantized_cache* c, Span (&spans)[4]) {
  const int64_t rows = c->pages * c->heads * c->page_size;
  spans[0] = Span{c->key_codes, rows * (c->dim / 2)};
  spans[1] = Span{c->value_codes, rows * (c->dim / 2)};
  spans[2] = Span{c->key_scales, rows * (c->dim / 8)};
  spans[3] = Span{c->value_scales, rows * (c->dim / 8)};
}

bool meets_pool(const rkv_quantized_cache* c, Span s) {
  Span spans[4];
  pool_spans(c, spans);
  for (const Span& p : spans)
    if (spans_meet(p, s)) return true;
  return false;
}

// (tokens, heads, dim) rows of 16-bit elements.
Span rows_span(const void* rows, int64_t token_stride, int64_t head_stride, int64_t tokens,
               int64_t heads, int64_t dim) {
  if (tokens <= 0 || heads <= 0) return Span{rows, 0};
  return Span{rows, 2 * ((tokens - 1) * token_stride + (heads - 1) * head_stride + dim)};
}

int check_quantized(const char* who, const rkv_quantized_cache* c) {
  const int64_t lim = (int64_t(1) << 31) - 1;
  if (!c) return set_error(kInvalidArgument, "%s: null cache", who);
  if (!c->key_codes || !c->value_codes || !c->key_scales || !c->value_scales ||
      !c->block_table || !c->lengths)
    return set_error(kInvalidArgument, "%s: null pointer in the cache", who);
  if (c->dtype != RKV_BF16 && c->dtype != RKV_F16)
    return set_error(kUnsupported, "%s: the rows must be bfloat16 or float16", who);
  if (!supported_dim(c->dim))
    return set_error(kUnsupported, "%s: head_dim %lld not in 32..256 step 32", who,
                     (long long)c->dim);
  if (c->pages <= 0 || c->heads <= 0 || c->sequences <= 0 || c->max_blocks <= 0 ||
      c->pages > lim || c->heads > 65535 || c->sequences > lim)
    return set_error(kInvalidArgument, "%s: empty or oversized cache", who);
  if (page_shift(c->page_size) < 0)
    return set_error(kUnsupported, "%s: page_size %lld not in {16, 32, 64, 128, 256}", who,
                     (long long)c->page_size);
  if (c->max_blocks > lim / c->page_size)
    return set_error(kInvalidArgument, "%s: the block table covers 2^31 tokens or more", who);
  if (c->table_stride < 0) return set_error(kInvalidArgument, "%s: negative stride", who);
  if (!aligned(c->key_codes, 16) || !aligned(c->value_codes, 16) || !aligned(c->key_scales, 16) ||
      !aligned(c->value_scales, 16))
    return set_error(kInvalidArgument, "%s: the cache must be 16-byte aligned", who);
  Span spans[4];
  pool_spans(c, spans);
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (spans_meet(spans[i], spans[j]))
        return set_error(kInvalidArgument, "%s: the cache's parts share memory", who);
  return kOk;
}

int check_tiles(const char* who, const rkv_quantized_cache* c, int64_t group) {
  if (group <= 0) return set_error(kInvalidArgument, "%s: empty group", who);
  if (group > kMaxGroup)
    return set_error(kUnsupported, "%s: GQA group %lld exceeds 16", who, (long long)group);
  // tiles and rows are counted in 32 bits
  const int64_t tiles = c->max_blocks * c->page_size / kTileTokens + 1;
  if (tiles > ((int64_t(1) << 31) - 1) / c->heads / c->sequences)
    return set_error(kUnsupported, "%s: the block table covers too many tokens", who);
  return kOk;
}

PagedPlan quantized_plan(const rkv_quantized_cache* c, int64_t group) {
  int grid = 0;
  RKV_DISPATCH_DIM(c->dim, D, grid = compute_units() * kPerCu4<D>);
  return plan_of(grid, group, c->dim);
}

// What append and read share: tokens, their sequences and the cache's places.
int rows_args(const char* who, QuantRows& a, const rkv_quantized_cache* c, int64_t tokens,
              const int32_t* token_starts) {
  if (tokens < 0 || (!token_starts && tokens != c->sequences))
    return set_error(kInvalidArgument, "%s: without token_starts one token per sequence", who);
  a.heads = (int)c->heads;
  a.tokens = tokens;
  a.dim = (int)c->dim;
  a.starts = token_starts;
  a.lengths = c->lengths;
  a.table = c->block_table;
  a.table_stride = c->table_stride;
  a.sequences = (int)c->sequences;
  a.max_blocks = (int)c->max_blocks;
  a.pages = (int)c->pages;
  a.shift = page_shift(c->page_size);
  a.keys = Pool{static_cast<char*>(c->key_codes), static_cast<char*>(c->key_scales)};
  a.values = Pool{static_cast<char*>(c->value_codes), static_cast<char*>(c->value_scales)};
  return kOk;
}

// Heads that a token's threads hold at a time, and the grid: `heads` rows a
// token, `items` threads a row.  Few tokens: all threads of a workgroup, for
// latency.
int rows_grid(const char* who, QuantRows& a, int heads, int items, int64_t& blocks) {
  a.slots = kRowThreads / items;
  if (a.tokens * items * a.slots >= kManyRowThreads) a.slots = items < kWave / 2 ? kWave / 2 / items : 1;
  a.slots = a.slots < heads ? a.slots : heads;
  a.per_block = kRowThreads / (items * a.slots);
  blocks = (a.tokens + a.per_block - 1) / a.per_block;
  return launch_fits(blocks, kRowThreads) ? kOk
                                          : set_error(kInvalidArgument, "%s: too many tokens", who);
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_quantized_append(const rkv_quantized_cache* cache, const void* query,
                                    int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                                    void* query_out, int64_t qo_token_stride,
                                    int64_t qo_head_stride, const void* key,
                                    int64_t k_token_stride, int64_t k_head_stride,
                                    const void* value, int64_t v_token_stride,
                                    int64_t v_head_stride, int64_t tokens,
                                    const int32_t* token_starts, const double* rates,
                                    int64_t rotary_dim, int interleaved, float scale,
                                    hipStream_t stream) {
  const char* who = "rkv_quantized_append";
  clear_error();
  int rc = check_quantized(who, cache);
  if (rc) return rc;
  QuantRows a{};
  rc = rows_args(who, a, cache, tokens, token_starts);
  if (rc) return rc;
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > cache->dim || (rotary_dim > 0 && !rates))
    return set_error(kInvalidArgument, "%s: rotary_dim %lld must be even, at most head_dim, with "
                     "its rates", who, (long long)rotary_dim);
  if (q_heads < 0 || q_heads > 65535)
    return set_error(kInvalidArgument, "%s: bad head count", who);
  if (tokens == 0) return kOk;
  const int64_t heads[3] = {q_heads, cache->heads, cache->heads};
  const void* src[3] = {query, key, value};
  const int64_t ts[3] = {q_token_stride, k_token_stride, v_token_stride};
  const int64_t hs[3] = {q_head_stride, k_head_stride, v_head_stride};
  for (int i = 0; i < 3; ++i) {
    if (!heads[i]) continue;
    a.src[i] = static_cast<const char*>(src[i]);
    a.src_ts[i] = read_stride(ts[i], tokens);
    a.src_hs[i] = read_stride(hs[i], heads[i]);
    if (!src[i]) return set_error(kInvalidArgument, "%s: null pointer argument", who);
    if (!aligned(src[i], 16) || a.src_ts[i] % 8 || a.src_hs[i] % 8 || a.src_ts[i] < 0 ||
        a.src_hs[i] < 0)
      return set_error(kInvalidArgument, "%s: rows must be 16-byte aligned with strides in "
                       "multiples of 8", who);
    if (meets_pool(cache, rows_span(src[i], a.src_ts[i], a.src_hs[i], tokens, heads[i],
                                    cache->dim)))
      return set_error(kInvalidArgument, "%s: rows overlap the cache", who);
  }
  if (q_heads) {
    a.dst[0] = static_cast<char*>(query_out);
    a.dst_ts = read_stride(qo_token_stride, tokens);
    a.dst_hs = read_stride(qo_head_stride, q_heads);
    if (!query_out) return set_error(kInvalidArgument, "%s: null pointer argument", who);
    if (!aligned(query_out, 16) || a.dst_ts % 8 || a.dst_hs % 8 || a.dst_ts < 0 || a.dst_hs < 0)
      return set_error(kInvalidArgument, "%s: query_out must be 16-byte aligned with strides in "
                       "multiples of 8", who);
    if (meets_pool(cache, rows_span(query_out, a.dst_ts, a.dst_hs, tokens, q_heads, cache->dim)))
      return set_error(kInvalidArgument, "%s: query_out overlaps the cache", who);
    // an item's partner dims are read from the row: it is not turned in place
    if (spans_meet(rows_span(query, a.src_ts[0], a.src_hs[0], tokens, q_heads, cache->dim),
                   rows_span(query_out, a.dst_ts, a.dst_hs, tokens, q_heads, cache->dim)))
      return set_error(kInvalidArgument, "%s: query_out overlaps the query", who);
  }
  a.q_heads = (int)q_heads;
  a.rotary_dim = (int)rotary_dim;
  a.interleaved = interleaved != 0;
  a.rates = rates;
  a.scale = scale;
  int64_t blocks;
  const bool halves = !a.interleaved && rotary_dim == cache->dim && rotary_dim / 2 % kGroupDims == 0;
  rc = rows_grid(who, a, a.q_heads + 2 * a.heads, a.dim / (halves ? 2 * kItem : kItem), blocks);
  if (rc) return rc;
  const dim3 grid((unsigned)blocks), threads(kRowThreads);
  const bool half = cache->dtype == RKV_F16;
  if (halves) {
    if (half) quantize_rows_kernel<_Float16, kHalves><<<grid, threads, 0, stream>>>(a);
    else quantize_rows_kernel<__bf16, kHalves><<<grid, threads, 0, stream>>>(a);
  } else if (a.interleaved || rotary_dim == 0) {
    if (half) quantize_rows_kernel<_Float16, kWithin><<<grid, threads, 0, stream>>>(a);
    else quantize_rows_kernel<__bf16, kWithin><<<grid, threads, 0, stream>>>(a);
  } else if (rotary_dim / 2 % kItem == 0) {
    if (half) quantize_rows_kernel<_Float16, kWhole><<<grid, threads, 0, stream>>>(a);
    else quantize_rows_kernel<__bf16, kWhole><<<grid, threads, 0, stream>>>(a);
  } else {
    if (half) quantize_rows_kernel<_Float16, kParts><<<grid, threads, 0, stream>>>(a);
    else quantize_rows_kernel<__bf16, kParts><<<grid, threads, 0, stream>>>(a);
  }
  return check_launch("quantize_rows_kernel");
}

extern "C" int rkv_quantized_read(const rkv_quantized_cache* cache, int64_t tokens,
                                  const int32_t* token_starts, void* key_out, void* value_out,
                                  hipStream_t stream) {
  const char* who = "rkv_quantized_read";
  clear_error();
  int rc = check_quantized(who, cache);
  if (rc) return rc;
  QuantRows a{};
  rc = rows_args(who, a, cache, tokens, token_starts);
  if (rc) return rc;
  if (tokens == 0) return kOk;
  if (!key_out || !value_out) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  if (!aligned(key_out, 16) || !aligned(value_out, 16))
    return set_error(kInvalidArgument, "%s: rows must be 16-byte aligned", who);
  const Span keys = rows_span(key_out, cache->heads * cache->dim, cache->dim, tokens, cache->heads,
                              cache->dim);
  const Span values{value_out, keys.bytes};
  if (meets_pool(cache, keys) || meets_pool(cache, values) || spans_meet(keys, values))
    return set_error(kInvalidArgument, "%s: the rows overlap each other or the cache", who);
  a.dst[1] = static_cast<char*>(key_out);
  a.dst[2] = static_cast<char*>(value_out);
  int64_t blocks;
  rc = rows_grid(who, a, 2 * a.heads, a.dim / kItem, blocks);
  if (rc) return rc;
  const dim3 grid((unsigned)blocks), threads(kRowThreads);
  if (cache->dtype == RKV_F16) quantized_read_kernel<_Float16><<<grid, threads, 0, stream>>>(a);
  else quantized_read_kernel<__bf16><<<grid, threads, 0, stream>>>(a);
  return check_launch("quantized_read_kernel");
}

extern "C" int rkv_quantized_plan(const rkv_quantized_cache* cache, int64_t group,
                                  size_t* workspace_bytes) {
  const char* who = "rkv_quantized_plan";
  clear_error();
  if (!workspace_bytes) return set_error(kInvalidArgument, "%s: null pointer", who);
  int rc = check_quantized(who, cache);
  if (!rc) rc = check_tiles(who, cache, group);
  if (rc) return rc;
  *workspace_bytes = quantized_plan(cache, group).total;
  return kOk;
}

extern "C" int rkv_quantized_decode(const rkv_quantized_cache* cache, const void* query,
                                    int64_t q_sequence_stride, int64_t q_head_stride,
                                    int64_t group, float scale, const rkv_scores* scores,
                                    void* output, void* workspace, size_t workspace_bytes,
                                    hipStream_t stream) {
  const char* who = "rkv_quantized_decode";
  clear_error();
  int rc = check_quantized(who, cache);
  if (!rc) rc = check_tiles(who, cache, group);
  if (rc) return rc;
  QuantArgs a{};
  rc = walk_args(who, a, *cache, query, q_sequence_stride, q_head_stride, group, scale, scores,
                 output);
  if (rc) return rc;
  if (meets_pool(cache, Span{output, cache->sequences * cache->heads * group * cache->dim * 2}))
    return set_error(kInvalidArgument, "%s: output overlaps the cache", who);
  const PagedPlan P = quantized_plan(cache, group);
  rc = use_workspace(who, a, P, workspace, workspace_bytes);
  if (rc) return rc;
  a.key_codes = static_cast<const char*>(cache->key_codes);
  a.key_scales = static_cast<const char*>(cache->key_scales);
  a.value_codes = static_cast<const char*>(cache->value_codes);
  a.value_scales = static_cast<const char*>(cache->value_scales);
  const dim3 grid((unsigned)P.grid), join((unsigned)P.grid, (unsigned)group);
  // (scores that are scaled late are scaled by a number above 0)
  const bool plain = !scores_any(scores) && a.scale != 0.0f && a.scale - a.scale == 0.0f;
  const size_t parts = part_bytes(group, cache->dim);
  RKV_DISPATCH_DIM(cache->dim, D, {
    if (cache->dtype == RKV_F16) {
      if (plain) quantized_kernel<D, true, false><<<grid, dim3(kThreads), parts, stream>>>(a);
      else quantized_kernel<D, true, true><<<grid, dim3(kThreads), parts, stream>>>(a);
      paged_join_kernel<D, true><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    } else {
      if (plain) quantized_kernel<D, false, false><<<grid, dim3(kThreads), parts, stream>>>(a);
      else quantized_kernel<D, false, true><<<grid, dim3(kThreads), parts, stream>>>(a);
      paged_join_kernel<D, false><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    }
  });
  return check_launch("quantized_kernel");
}
