// What the decodes over a paged cache share (rkv_paged.hip, 16-bit pages;
// rkv_quantized.hip, 4-bit ones): every wave's share of all sequences' tiles,
// the walk over them, the softmax, and the join of rows that several waves and
// workgroups hold parts of.  How a tile is loaded and multiplied is the
// store's (Pages16, Pages4).
#pragma once

#include <atomic>
#include <type_traits>

#include "rkv_common.h"
#include "rkv_internal.h"
#include "rkv_paged.h"

namespace rkv {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kJoinThreads = 256;
constexpr int kTileTokens = 32;  // tokens a wave takes at a time: two halves of 16

// Workgroups' entries of WalkArgs::open, a cache line apart: the join's
// workgroup k runs on the XCD of the attention's and finds its own line in
// that L2 (one sequence of 2003 tokens 12.0 -> 11.75 us).
constexpr int kOpenStride = 16;

typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef float F32x4 __attribute__((ext_vector_type(4)));

// A type's matrix products (16 x 16 x 32) and its rounding of pairs.
template <bool kHalf>
struct Type16;
template <>
struct Type16<false> {
  typedef __bf16 E;
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ F32x4 mma(V8 a, V8 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Type16<true> {
  typedef _Float16 E;
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ F32x4 mma(V8 a, V8 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

struct WalkArgs {
  const char* query;             // (B, H G, D), strides in elements
  int64_t q_bs, q_hs;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int sequences, heads, group, max_blocks, pages, shift;
  float scale;                   // times log2 e: the softmax runs on 2^x
  char* out;                     // (B, H G, D) dense
  // a row (sequence, KV head) whose tiles lie in several workgroups: their
  // partial results, [workgroup][0: began before, 1: begins here]
  int2* open;                    // [workgroup]: the row that begins there (-1: none goes on
                                 // behind it), the workgroups that hold parts of it
  float2* part_ml;               // [..][group]
  float* part_acc;               // [..][group][D]
  // scores that are more than products (kScores)
  float cap, per_cap;            // > 0: s = cap tanh(s / cap); cap times log2 e, scale / cap
  const float* slopes;           // [H G]: s -= slope * distance (null: none)
  int window;                    // tokens up to this one that are seen
};

// Dims of a value row that a lane holds: D / 16 of them, as 16-, 8- and
// 4-byte pieces (of 128, 64 and 32 dims of the row).
template <int D>
struct Pieces {
  static constexpr int k8 = D / 128;
  static constexpr int k4 = D % 128 >= 64 ? 1 : 0;
  static constexpr int k2 = D % 64 >= 32 ? 1 : 0;
  static constexpr int kBlocks = D / 16;  // 16-dim matrix products: 8 k8 + 4 k4 + 2 k2
  // Calls put(first product, first dim, size as an integral constant) for each
  // piece of lane column i: the products' dims are consecutive there.
  template <typename Put>
  static __device__ __forceinline__ void each(int i, Put put) {
#pragma unroll
    for (int c = 0; c < k8; ++c) put(8 * c, 128 * c + i * 8, std::integral_constant<int, 8>());
    if constexpr (k4 > 0) put(8 * k8, 128 * k8 + i * 4, std::integral_constant<int, 4>());
    if constexpr (k2 > 0)
      put(8 * k8 + 4 * k4, 128 * k8 + 64 * k4 + i * 2, std::integral_constant<int, 2>());
  }
};

// A buffer view of `bytes` bytes at `base`, both wave-uniform; loads past it
// return zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t view_of(const char* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo),
                                           (short)0, (int)__builtin_amdgcn_readfirstlane(bytes),
                                           0x00020000);
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// An int of an array that does not change during a launch, at a wave-uniform
// place: a scalar load.
__device__ __forceinline__ int scalar_at(const int32_t* p, int64_t i) {
  typedef __attribute__((address_space(4))) const int32_t ConstI32;
  return ((ConstI32*)(uintptr_t)p)[i];
}

// A sequence's length as attended: negative is 0; one past the table is 0 with
// its row marked bad.
__device__ __forceinline__ int length_of(const WalkArgs& a, int n, bool& bad) {
  bad = n > 0 && (n - 1) >> a.shift >= a.max_blocks;
  return bad || n < 0 ? 0 : n;
}

// Inclusive sum over the wave's lanes: within rows of 16 by row shifts, then
// the rows' totals.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  const int lane = threadIdx.x % kWave;
#define SHR(n) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x110 + n, 0xF, 0xF, false)
  SHR(1);
  SHR(2);
  SHR(4);
  SHR(8);
#undef SHR
  const uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)x, 15);
  const uint32_t r1 = r0 + (uint32_t)__builtin_amdgcn_readlane((int)x, 31);
  const uint32_t r2 = r1 + (uint32_t)__builtin_amdgcn_readlane((int)x, 47);
  return x + (lane < 16 ? 0u : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

// The first tile of a sequence's row that holds a visible token.
template <bool kScores>
__device__ __forceinline__ int first_of(const WalkArgs& a, int length) {
  return kScores && length > a.window ? (length - a.window) / kTileTokens : 0;
}

// The tile behind a sequence's last: the first one at least, so that every row
// has an owner that writes its output.
__device__ __forceinline__ int tiles_of(int length) {
  return length > kTileTokens ? (length - 1) / kTileTokens + 1 : 1;
}

// Where a wave stands in the list of all tiles: sequence by sequence, KV head
// by KV head, tile by tile.
struct Cursor {
  int b, h, tile, tiles, length;
  int first;         // (kScores) the row's first tile
  int page0, page1;  // of the tile's two halves, as the table has them
  bool bad;
};

template <bool kScores>
__device__ __forceinline__ int first_tile(const Cursor& c) {
  return kScores ? c.first : 0;
}

template <bool kScores>
__device__ __forceinline__ void begin_sequence(const WalkArgs& a, Cursor& c) {
  c.length = length_of(a, scalar_at(a.lengths, c.b), c.bad);
  c.tiles = tiles_of(c.length);
  if constexpr (kScores) c.first = first_of<kScores>(a, c.length);
}

// The table's entries for the tile (any in-bounds entry for a half with no
// token, whose page is not used).
__device__ __forceinline__ void fetch_pages(const WalkArgs& a, Cursor& c) {
  const int t0 = c.tile * kTileTokens, t1 = t0 + kTileTokens / 2;
  const int64_t row = (int64_t)c.b * a.table_stride;
  c.page0 = scalar_at(a.table, row + (t0 < c.length ? t0 >> a.shift : 0));
  c.page1 = scalar_at(a.table, row + (t1 < c.length ? t1 >> a.shift : 0));
}

template <bool kScores>
__device__ __forceinline__ void next_tile(const WalkArgs& a, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = first_tile<kScores>(c);
  if (++c.h < a.heads) return;
  c.h = 0;
  if (c.b + 1 < a.sequences) {
    ++c.b;
    begin_sequence<kScores>(a, c);
    c.tile = first_tile<kScores>(c);
  }
}

struct PartHead {
  int row;              // -1: unused
  int begins, ends;     // the row's first / last tile is in the wave
  uint32_t from, tiles;  // the row's tiles in the list of all
};

// The (begin, count) of a wave's tiles in the list of all: an equal share each,
// the first `extra` waves one more.
struct Shares {
  uint32_t share, extra;
  __device__ __forceinline__ uint32_t begin(uint32_t id) const {
    return id * share + (id < extra ? id : extra);
  }
  __device__ __forceinline__ uint32_t workgroup_of(uint32_t tile) const {
    const uint32_t longer = extra * (share + 1u);
    return (tile < longer ? tile / (share + 1u) : extra + (tile - longer) / share) / kWaves;
  }
};

// Folds parts j = first, first + step, .. of n into (m, l, o): in batches whose
// loads are all in flight before the first use.  kKeep: infinite and NaN sums
// count whatever their part weighs (else one that weighs 0 is NaN).
template <bool kKeep = false, typename Ml, typename Acc>
__device__ __forceinline__ void fold_parts(uint32_t first, uint32_t step, uint32_t n, float& m,
                                           float& l, F32x4& o, Ml load_ml, Acc load_acc) {
  constexpr uint32_t kBatch = 8;
  auto weighed = [](F32x4 x, float w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = kKeep && !__builtin_isfinite(x[i]) ? x[i] : x[i] * w;
    return x;
  };
  for (uint32_t j0 = first; j0 < n; j0 += step * kBatch) {
    float2 ml[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const uint32_t j = min(j0 + i * step, n - 1u);
      ml[i] = load_ml(j);
      x[i] = load_acc(j);
    }
    float mn = m;
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) mn = __builtin_fmaxf(mn, ml[i].x);
    const float old = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    l *= old;
    o = weighed(o, old);
    m = mn;
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const bool there = j0 + i * step < n;
      const float w = ml[i].x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - mn);
      // (a NaN sum stays one, whatever its weight)
      l += there ? ml[i].y * w : 0.0f;
      o += there ? weighed(F32x4{x[i].x, x[i].y, x[i].z, x[i].w}, w)
                 : F32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
}

// tanh: by its series up to 1/4 (the next term is 1e-8 of it), then by e^2y on
// the hardware's transcendental unit, off by some 2^-22 absolute.
__device__ __forceinline__ float tanh_hw(float y) {
  const float y2 = y * y;
  float s = 2.18694885361552028e-02f;                    // 62/2835
  s = __builtin_fmaf(s, y2, -5.39682539682539683e-02f);  // 17/315
  s = __builtin_fmaf(s, y2, 1.33333333333333333e-01f);   // 2/15
  s = __builtin_fmaf(s, y2, -3.33333333333333333e-01f);  // 1/3
  const float near = __builtin_fmaf(s * y2, y, y);
  const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
  return __builtin_fabsf(y) < 0.25f ? near : far;
}

// Every wave takes an equal, contiguous share of all tiles and walks it alone:
// the keys and values of the next tile are loading while one is computed,
// across rows' ends too, so that ragged batches stream like long ones.  A
// tile's S^T = K Q^T and O^T = V^T P^T run on the matrix cores with the query
// rows in the columns, so that a lane's maximum, sum and accumulators all
// belong to query row l % 16:
//   S^T: A = 16 key rows straight from memory (lane l: row l % 16, dims
//     8 (l / 16) + 32 j ..), B = the query rows; the result in lane l is
//     S[t = 4 (l / 16) + r][l % 16], r = 0..3.
//   O^T: B = P^T, whose k slots 8 (l / 16) + e are tokens 4 (l / 16) + e of
//     the first half (e < 4) and 4 (l / 16) + e - 4 of the second: the values
//     that lane l already holds.  A = V^T over the same slots: lane l loads
//     the same 8 dims of those 8 tokens (16 lanes: a whole row) and
//     transposes them with byte permutes; the m-th of 8 products takes dim
//     8 (l % 16) + m for its row l % 16.  (Rows of 64 and 32 dims: 4 and 2.)
template <typename Store, bool kScores>
__device__ __forceinline__ void walk(const typename Store::Args& a) {
  constexpr int D = Store::kDim;
  using E = typename Type16<Store::kHalf>::E;
  using P = Pieces<D>;
  using Tile = typename Store::Tile;
  // a wave's results of rows that it does not hold whole: [wave][0: the row
  // began before, 1: it begins here]
  extern __shared__ float4 lds[];
  float* const part_acc = reinterpret_cast<float*>(lds);  // [part][group][D]
  float2* const part_ml = reinterpret_cast<float2*>(part_acc + kWaves * 2 * a.group * D);
  __shared__ PartHead heads_s[kWaves][2];
  __shared__ float weight_s[kMaxGroup][16];
  __shared__ float2 total_s[kMaxGroup];
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = uniform(tid / kWave);
  const int li = lane & 15, lg = lane >> 4;
  if (tid < kWaves * 2) heads_s[tid / 2][tid % 2].row = -1;
  __syncthreads();

  // ---- this wave's share of the tiles: every wave sums the lengths itself,
  // each lane those of `per` sequences (no exchange between waves)
  const int per = (a.sequences + kWave - 1) / kWave;
  const int b0 = lane * per;
  uint32_t sum = 0;
#pragma unroll 4
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    bool bad;
    const int length = length_of(a, a.lengths[b < a.sequences ? b : a.sequences - 1], bad);
    const int n = tiles_of(length) - first_of<kScores>(a, length);
    sum += b < a.sequences ? (uint32_t)n : 0u;
  }
  sum *= (uint32_t)a.heads;
  const uint32_t upto = wave_scan(sum);  // tiles up to the lane's last sequence
  const uint32_t total = (uint32_t)uniform((int)__shfl((int)upto, kWave - 1, kWave));
  uint32_t waves = gridDim.x * kWaves;
  waves = total < waves ? total : waves;
  const uint32_t id = blockIdx.x * kWaves + (uint32_t)wave;
  const Shares shares{total / waves, total % waves};
  uint32_t left = id < waves ? shares.share + (id < shares.extra ? 1u : 0u) : 0u;
  if (left > 0) {
    const uint32_t start = shares.begin(id);
    uint32_t pos = start;  // the computed tile's place in the list
    const uint64_t after = __builtin_amdgcn_ballot_w64(upto > start);
    const int owner = (int)__builtin_ctzll(after);  // the lane whose sequences hold the start
    uint32_t rest = start - (uint32_t)uniform(__shfl((int)(upto - sum), owner, kWave));
    Cursor cur;
    cur.b = owner * per;
    for (;; ++cur.b) {
      begin_sequence<kScores>(a, cur);
      const uint32_t here = (uint32_t)(cur.tiles - first_tile<kScores>(cur)) * (uint32_t)a.heads;
      if (rest < here || cur.b + 1 >= a.sequences) break;
      rest -= here;
    }
    const uint32_t count = (uint32_t)(cur.tiles - first_tile<kScores>(cur));
    cur.h = (int)(rest / count);
    cur.tile = (int)(rest % count) + first_tile<kScores>(cur);
    fetch_pages(a, cur);

    const Store store(a, li, lg);
    F32x4 acc[Store::kAccs];
    typename Store::Query q;
    U32x4 q_next[D / 32];  // the next row's, loading with its first tile
    float slope = 0.0f, slope_next = 0.0f;  // (kScores) of the lane's query row, times log2 e
    float m = kNegInf, l = 0.0f;
    bool bad_row = false;
    bool begun = false;  // the row's first tile was this wave's

    // (query rows past the group read outside the view: zeros)
    const uint32_t qo = li < a.group ? (uint32_t)li * (uint32_t)a.q_hs * 2u + (uint32_t)lg * 16u
                                     : 0x80000000u;
    auto load_query = [&](const Cursor& c) {
      const auto qr = view_of(
          a.query + ((int64_t)c.b * a.q_bs + (int64_t)c.h * a.group * a.q_hs) * 2,
          (uint32_t)(a.group - 1) * (uint32_t)a.q_hs * 2u + D * 2u);
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        q_next[j] = __builtin_amdgcn_raw_buffer_load_b128(qr, (int)(qo + 64u * j), 0, 0);
      if constexpr (kScores)
        if (a.slopes) slope_next = a.slopes[c.h * a.group + min(li, a.group - 1)];
    };

    auto begin_row = [&](const Cursor& c) {
      store.take(q, q_next);
      if constexpr (kScores) slope = slope_next * kLog2e;
#pragma unroll
      for (int n = 0; n < Store::kAccs; ++n) acc[n] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m = kNegInf;
      l = 0.0f;
      bad_row = false;
      begun = c.tile == first_tile<kScores>(c);
    };

    auto compute = [&](const Cursor& c, Tile& t, bool bad, bool last_tile) {
      bad_row |= bad;
      {
        float x[8];
        store.scores(q, t, x);
        // tokens of the tile that are seen: those behind the sequence's end, and
        // (kScores) those before the window, weigh nothing
        const int behind = c.length - c.tile * kTileTokens;
        const int from = kScores ? behind - a.window : 0;
        auto token = [&](int e) { return 16 * (e / 4) + 4 * lg + e % 4; };
        if constexpr (kScores) {
          const float by = store.unit(q) * (a.cap > 0.0f ? a.per_cap : a.scale);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= by;
          if (a.cap > 0.0f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = tanh_hw(x[e]) * a.cap;
          }
          if (a.slopes) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] -= slope * (float)(behind - 1 - token(e));
          }
        } else if constexpr (!Store::kScaleLate) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= a.scale;
        }
        if (behind < kTileTokens) {
          if constexpr (Store::kRareEnds) asm volatile("");
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = token(e) < behind ? x[e] : kNegInf;
        }
        if (kScores && from > 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = token(e) >= from ? x[e] : kNegInf;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, x[e]);
        float u, w;
        xor16_pair(top, u, w);
        top = __builtin_fmaxf(u, w);
        xor32_pair(top, u, w);
        top = __builtin_fmaxf(u, w);
        // (kScaleLate: the scores are multiplied on the way into the exponential)
        constexpr bool kLate = Store::kScaleLate && !kScores;
        // (never 0: a hidden score times it would be NaN)
        const float late =
            kLate ? __builtin_fmaxf(store.unit(q) * a.scale, __FLT_MIN__) : 1.0f;
        if constexpr (kLate) top *= late;
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float mn = __builtin_fmaxf(m, top);
          const float by = mn == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= by;
#pragma unroll
          for (int n = 0; n < Store::kAccs; ++n) acc[n] *= by;
        }
        const float base = m == kNegInf ? 0.0f : m;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // (fp16 weights go up to 2^15 instead of 1, and the sum with them, so
          // that those of 2^-24 to 2^-39 of the largest, many in a long
          // context, do not round to zero)
          if constexpr (Store::kScaleLate)
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], late, 15.0f - base));
          else
            p[e] = __builtin_amdgcn_exp2f(x[e] - base) * (Store::kHalf ? 32768.0f : 1.0f);
          l += p[e];
        }
        store.products(acc, t, p, from, behind);
      }
      const bool ends = c.tile + 1 == c.tiles;
      if (!ends && !last_tile) return;
      store.finish(acc);
      float u, w, sum_l = l;
      xor16_pair(sum_l, u, w);
      sum_l = u + w;
      xor32_pair(sum_l, u, w);
      sum_l = u + w;
      if (bad_row) sum_l = __builtin_nanf("");
      const int row = c.b * a.heads + c.h;
      if (begun && ends) {
        if (li < a.group) {
          // a sequence without tokens gives zeros
          const float by = c.length == 0 && !bad_row ? 0.0f : 1.0f / sum_l;
          char* out = a.out + ((int64_t)row * a.group + li) * (D * 2);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            P::each(4 * lg + r, [&](int n0, int d, auto size) {
              typedef E EN __attribute__((ext_vector_type(size())));
              EN y;
#pragma unroll
              for (int i = 0; i < size(); ++i) y[i] = (E)(acc[n0 + i][r] * by);
              *reinterpret_cast<EN*>(out + d * 2) = y;
            });
        }
        return;
      }
      const int slot = begun ? 1 : 0;
      const int part = (wave * 2 + slot) * a.group;
      if (lane == 0) {
        const uint32_t first = (uint32_t)first_tile<kScores>(c);
        heads_s[wave][slot] = PartHead{row, begun, ends, pos - ((uint32_t)c.tile - first),
                                       (uint32_t)c.tiles - first};
      }
      if (li < a.group) {
        if (lg == 0) part_ml[part + li] = make_float2(m, sum_l);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          P::each(4 * lg + r, [&](int n0, int d, auto size) {
            constexpr int kN = size() < 4 ? size() : 4;
            typedef float FN __attribute__((ext_vector_type(kN)));
#pragma unroll
            for (int i = 0; i < size(); i += kN) {
              FN y;
#pragma unroll
              for (int j = 0; j < kN; ++j) y[j] = acc[n0 + i + j][r];
              *reinterpret_cast<FN*>(&part_acc[(part + li) * D + d + i]) = y;
            }
          });
      }
    };

    Tile t0, t1;
    Cursor ahead = cur, far;  // the tile that is loading, and the one after it
    load_query(cur);
    bool bad0 = store.load(cur, t0, true), bad1 = false;
    if (left > 1) {
      next_tile<kScores>(a, ahead);
      fetch_pages(a, ahead);
    }
    bool row_start = true;  // of the row, or of the wave's share of it
    auto step = [&](Tile& now, bool bad, Tile& next) -> bool {
      if (row_start) begin_row(cur);
      if (left > 1 && ahead.tile == first_tile<kScores>(ahead)) load_query(ahead);
      far = ahead;
      if (left > 2) {
        next_tile<kScores>(a, far);
        fetch_pages(a, far);
      }
      const bool next_bad = store.load(ahead, next, left > 1);
      compute(cur, now, bad, left == 1);
      cur = ahead;
      ahead = far;
      row_start = cur.tile == first_tile<kScores>(cur);
      ++pos;
      return next_bad;
    };
    for (;;) {
      bad1 = step(t0, bad0, t1);
      if (--left == 0) break;
      bad0 = step(t1, bad1, t0);
      if (--left == 0) break;
    }
  }
  __syncthreads();

  // ---- the waves' parts of rows: neighbours of one row are joined, in order
  if (tid == 0) a.open[blockIdx.x * kOpenStride] = make_int2(-1, 0);
  constexpr int kParts = 2 * kWaves;
  const PartHead mine = heads_s[lane % kParts / 2][lane % 2];  // lane i: part i
  const int my_row = lane < kParts ? mine.row : -1;
  uint64_t todo = __builtin_amdgcn_ballot_w64(my_row >= 0);
  while (todo) {
    const int first = (int)__builtin_ctzll(todo);
    const int row = __builtin_amdgcn_readlane(my_row, first);
    const uint64_t same = __builtin_amdgcn_ballot_w64(my_row == row);
    const int last = 63 - (int)__builtin_clzll(same), end = last + 1;
    const bool begins = __builtin_amdgcn_readlane(mine.begins, first);
    const bool ends = __builtin_amdgcn_readlane(mine.ends, last);
    todo &= ~same;
    const bool whole = begins && ends;
    const int to = blockIdx.x * 2 + (begins ? 1 : 0);
    // weights: lane i of 16 the row's part i of query row tid / 16
    for (int at = tid; at < kMaxGroup * 16; at += kThreads) {
      const int g = at / 16, i = at % 16;
      const bool in = same >> i & 1;
      const float2 ml =
          in && g < a.group ? part_ml[i * a.group + g] : make_float2(kNegInf, 0.0f);
      float M = ml.x;
      M = __builtin_fmaxf(M, row_ror<8>(M));
      M = __builtin_fmaxf(M, row_ror<4>(M));
      M = __builtin_fmaxf(M, row_ror<2>(M));
      M = __builtin_fmaxf(M, row_ror<1>(M));
      const float w = ml.x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
      // (a NaN sum stays one, whatever its weight)
      const float L = row16_sum_all(ml.y * w);
      weight_s[g][i] = w;
      if (i == 0) total_s[g] = make_float2(M, L);
    }
    __syncthreads();
    for (int x = tid; x < a.group * (D / 4); x += kThreads) {
      const int g = x / (D / 4), d = x % (D / 4) * 4;
      F32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int i = first; i < end; ++i) {
        const float w = weight_s[g][i];
        const F32x4 p = *reinterpret_cast<const F32x4*>(&part_acc[(i * a.group + g) * D + d]);
        // (a part that is not the row's holds anything)
        o += same >> i & 1 ? p * w : F32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
      const float2 ml = total_s[g];
      if (whole) {
        typedef E E4 __attribute__((ext_vector_type(4)));
        const float by = 1.0f / ml.y;
        E4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = (E)(o[r] * by);
        *reinterpret_cast<E4*>(a.out + (((int64_t)row * a.group + g) * D + d) * 2) = y;
      } else {
        const int64_t at = (int64_t)to * a.group + g;
        *reinterpret_cast<F32x4*>(a.part_acc + at * D + d) = o;
        if (d == 0) a.part_ml[at] = ml;
      }
    }
    if (begins && !ends && tid == 0) {
      const uint32_t from = (uint32_t)__builtin_amdgcn_readlane((int)mine.from, first);
      const uint32_t tiles = (uint32_t)__builtin_amdgcn_readlane((int)mine.tiles, first);
      const uint32_t to_last = shares.workgroup_of(from + tiles - 1u);
      a.open[blockIdx.x * kOpenStride] = make_int2(row, (int)(to_last - blockIdx.x + 1u));
    }
    if (todo) __syncthreads();
  }
}

// Joins the parts of one row that several workgroups hold: workgroup (k, g)
// query row g of the row that begins in the attention's workgroup k and goes
// on in those after it.
template <int D, bool kHalf>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(WalkArgs a) {
  constexpr int kStripes = kJoinThreads / (D / 4);
  __shared__ alignas(16) float acc_s[kStripes][D];
  __shared__ float2 ml_s[kStripes];
  const int k = blockIdx.x, g = blockIdx.y;
  const int2 held = a.open[k * kOpenStride];
  const int row = held.x, n = held.y;
  if (row < 0) return;
  const int c = threadIdx.x % (D / 4), stripe = threadIdx.x / (D / 4);
  float m = kNegInf, l = 0.0f;
  F32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (stripe < kStripes) {
    auto part_at = [&](uint32_t j) {
      return (2 * ((int64_t)k + j) + (j == 0 ? 1 : 0)) * a.group + g;
    };
    fold_parts((uint32_t)stripe, (uint32_t)kStripes, (uint32_t)n, m, l, o,
               [&](uint32_t j) { return a.part_ml[part_at(j)]; },
               [&](uint32_t j) {
                 return *reinterpret_cast<const float4*>(a.part_acc + part_at(j) * D + 4 * c);
               });
    *reinterpret_cast<F32x4*>(&acc_s[stripe][4 * c]) = o;
    if (c == 0) ml_s[stripe] = make_float2(m, l);
  }
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int d = threadIdx.x;
  float M = kNegInf, L = 0.0f, y = 0.0f;
  for (int j = 0; j < kStripes; ++j) M = __builtin_fmaxf(M, ml_s[j].x);
  for (int j = 0; j < kStripes; ++j) {
    const float w = ml_s[j].x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml_s[j].x - M);
    L += ml_s[j].y * w;
    y += acc_s[j][d] * w;
  }
  using E = typename Type16<kHalf>::E;
  *reinterpret_cast<E*>(a.out + (((int64_t)row * a.group + g) * D + d) * 2) = (E)(y / L);
}

// Compute units of the current device, 256 if unknown.
int compute_units() {
  static std::atomic<int> of_dev[64];  // per device; 0 = not asked yet
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = of_dev[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        n <= 0)
      return 256;
    of_dev[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

struct PagedPlan {
  int grid = 0;
  size_t ml_off = 0, acc_off = 0, total = 0;
};

PagedPlan plan_of(int grid, int64_t group, int64_t dim) {
  PagedPlan P;
  P.grid = grid;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t parts = (size_t)P.grid * 2;
  P.ml_off = up(P.grid * kOpenStride * sizeof(int2));
  P.acc_off = P.ml_off + up(parts * group * sizeof(float2));
  P.total = P.acc_off + up(parts * group * dim * sizeof(float));
  return P;
}

// Bytes of LDS that the walk's parts take.
size_t part_bytes(int64_t group, int64_t dim) {
  return (size_t)(kWaves * 2 * group) * (dim * sizeof(float) + sizeof(float2));
}

// The parts of a call's arguments that do not depend on how the cache holds its
// tokens: the query's and output's checks, the cache's tables (of either kind
// of cache), the scores.
template <typename Cache>
int walk_args(const char* who, WalkArgs& a, const Cache& cache, const void* query,
              int64_t q_sequence_stride, int64_t q_head_stride, int64_t group, float scale,
              const rkv_scores* scores, void* output) {
  if (!query || !output) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  q_sequence_stride = read_stride(q_sequence_stride, cache.sequences);
  q_head_stride = read_stride(q_head_stride, cache.heads * group);
  if (q_sequence_stride < 0 || q_head_stride < 0 || q_head_stride > (1 << 25))
    return set_error(kUnsupported, "%s: query stride", who);
  if (!aligned(query, 16) || !aligned(output, 16) || q_sequence_stride % 8 || q_head_stride % 8)
    return set_error(kInvalidArgument,
                     "%s: query and output must be 16-byte aligned with strides in multiples of 8",
                     who);
  const int rc = check_scores(who, scores);
  if (rc) return rc;
  a.query = static_cast<const char*>(query);
  a.q_bs = q_sequence_stride;
  a.q_hs = q_head_stride;
  a.table = cache.block_table;
  a.table_stride = cache.table_stride;
  a.lengths = cache.lengths;
  a.sequences = (int)cache.sequences;
  a.heads = (int)cache.heads;
  a.group = (int)group;
  a.max_blocks = (int)cache.max_blocks;
  a.pages = (int)cache.pages;
  a.shift = page_shift(cache.page_size);
  a.scale = scale * kLog2e;
  a.out = static_cast<char*>(output);
  a.window = scores_window(scores);
  if (scores) {
    a.slopes = scores->slopes;
    if (scores->softcap > 0.0f) {
      a.cap = scores->softcap * kLog2e;
      a.per_cap = scale / scores->softcap;
    }
  }
  return kOk;
}

int use_workspace(const char* who, WalkArgs& a, const PagedPlan& P, void* workspace,
                  size_t workspace_bytes) {
  if (!workspace || workspace_bytes < P.total)
    return set_error(kWorkspaceTooSmall, "%s: workspace of %zu bytes, %zu needed", who,
                     workspace_bytes, P.total);
  if (!aligned(workspace, 16))
    return set_error(kInvalidArgument, "%s: workspace must be 16-byte aligned", who);
  char* ws = static_cast<char*>(workspace);
  a.open = reinterpret_cast<int2*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + P.ml_off);
  a.part_acc = reinterpret_cast<float*>(ws + P.acc_off);
  return kOk;
}

}  // namespace
}  // namespace rkv
