// Attention of one new token per sequence over a paged KV cache:
//   out[b, h, g] = softmax_t(scale q[b, h, g] . K[t]) V,  t < lengths[b],
// token t of KV head h at row t % P of page table[b][t / P].
//
// Two launches: paged_kernel attends, paged_join_kernel joins the rows that
// several workgroups hold parts of.  (One launch whose last workgroup of a row
// joined it, through counters and stores past the caches, was as fast at best:
// one sequence of 2003 tokens 13.0 us against 12.5, of 131072 91.4 against
// 91.8, 128 short ones at head_dim 64 75 against 72.)  Sums, maxima and
// accumulators are fp32; the partition into shares depends on the batch's
// lengths and the device alone, so a call repeats bit for bit.
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

// Workgroups per CU that share the tiles.  One keeps the CU's loads full (each
// of its waves has two tiles on their way) and leaves the fewest parts to
// join; at head_dim 32 a tile is 4 KB and two are needed.  From one to two: 32,
// 64 sequences of up to 20000 tokens 157 -> 129.5 us; 64, 128 of up to 2000
// 72.5 -> 72.2; 96, 32 of up to 8000 85.9 -> 87.9; 128, 131072 tokens 92.4 ->
// 94.0; 160, 24 of up to 4000 61.3 -> 67.7.
template <int D>
constexpr int kPerCu = D < 64 ? 2 : 1;

// Workgroups' entries of PagedArgs::open, a cache line apart: the join's
// workgroup k runs on the XCD of the attention's and finds its own line in
// that L2 (one sequence of 2003 tokens 12.0 -> 11.75 us).
constexpr int kOpenStride = 16;

// Cache policy of the key and value loads: non-temporal.  A token is read once
// a step, and kept lines only push out others: 16 x 131072 tokens 1465 -> 1322
// us, one 103.5 -> 92.4, 64 ragged ones 111 -> 99.  (Sequences that share most
// of their pages lose what the caches would have held: 16 on the same 32768
// tokens 156 -> 206 us, 172 -> 276 on another card, 64 on the same 4096 79 ->
// 82; the host, which picks the kernel, does not know.)
constexpr int kStreamLoad = 2;
// That of a row's last 32 value dims, which lie in the half of a 128-byte line:
// kept where other loads take the rest of the line (head_dim 96, 32 x 8000
// tokens, 85.8 us against 87.2 non-temporal, 160 81.9 against 83.8, 224 82.2
// against 83.2), non-temporal where there are no others (head_dim 32, 64
// sequences of up to 20000 tokens, 129.4 against 134).
template <int D>
constexpr int kTailLoad = D == 32 ? kStreamLoad : 0;

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

struct PagedArgs {
  const char* query;             // (B, H G, D), strides in elements
  int64_t q_bs, q_hs;
  const char* keys;
  const char* values;
  int64_t k_ps, k_hs, v_ps, v_hs;  // page and head strides, elements
  uint32_t k_ts, v_ts;             // row strides, bytes
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

// One tile's operands as they come from memory.
template <int D>
struct Tile {
  using P = Pieces<D>;
  U32x4 k[2][D / 32];
  U32x4 v8[P::k8 ? P::k8 : 1][8];
  U32x2 v4[8];
  uint32_t v2[8];
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
__device__ __forceinline__ int length_of(const PagedArgs& a, int n, bool& bad) {
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

// Tiles of a sequence's row: one at least, so that every row has an owner
// that writes its output.
__device__ __forceinline__ int tiles_of(int length) {
  return length > kTileTokens ? (length - 1) / kTileTokens + 1 : 1;
}

// Where a wave stands in the list of all tiles: sequence by sequence, KV head
// by KV head, tile by tile.
struct Cursor {
  int b, h, tile, tiles, length;
  int page0, page1;  // of the tile's two halves, as the table has them
  bool bad;
};

// The table's entries for the tile (any in-bounds entry for a half with no
// token, whose page is not used).
__device__ __forceinline__ void fetch_pages(const PagedArgs& a, Cursor& c) {
  const int t0 = c.tile * kTileTokens, t1 = t0 + kTileTokens / 2;
  const int64_t row = (int64_t)c.b * a.table_stride;
  c.page0 = scalar_at(a.table, row + (t0 < c.length ? t0 >> a.shift : 0));
  c.page1 = scalar_at(a.table, row + (t1 < c.length ? t1 >> a.shift : 0));
}

__device__ __forceinline__ void next_tile(const PagedArgs& a, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.h < a.heads) return;
  c.h = 0;
  if (c.b + 1 < a.sequences) {
    ++c.b;
    c.length = length_of(a, scalar_at(a.lengths, c.b), c.bad);
    c.tiles = tiles_of(c.length);
  }
}

// A wave's results of a row that it does not hold whole.
template <int D>
struct Part {
  float acc[kMaxGroup][D];
  float2 ml[kMaxGroup];
};

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
// loads are all in flight before the first use.
template <typename Ml, typename Acc>
__device__ __forceinline__ void fold_parts(uint32_t first, uint32_t step, uint32_t n, float& m,
                                           float& l, F32x4& o, Ml load_ml, Acc load_acc) {
  constexpr uint32_t kBatch = 8;
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
    o *= old;
    m = mn;
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const bool there = j0 + i * step < n;
      const float w = ml[i].x == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - mn);
      // (a NaN sum stays one, whatever its weight)
      l += there ? ml[i].y * w : 0.0f;
      o += there ? F32x4{x[i].x, x[i].y, x[i].z, x[i].w} * w : F32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
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
// HBM bounds it: 8.6 GB of 16 x 131072 tokens (8 KV heads, group 4, d 128) in
// 1250-1325 us, 6.5-6.9 TB/s, by the card; the matrix cores are at 10 % and the
// vector ALUs at 15 %.  Small calls are a chain of latencies: 504 tiles of
// 2003 tokens take 7.2 us, of which 1.4 to know the share and its pages, 2.6
// until the first tile is done, 1.4 to join the waves; then 4.6 for the join
// kernel.
template <int D, bool kHalf>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void paged_kernel(PagedArgs a) {
  using T = Type16<kHalf>;
  using V8 = typename T::V8;
  using E = typename T::E;
  using P = Pieces<D>;
  __shared__ alignas(16) Part<D> parts[kWaves][2];
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
    const int n = tiles_of(length_of(a, a.lengths[b < a.sequences ? b : a.sequences - 1], bad));
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
      cur.length = length_of(a, scalar_at(a.lengths, cur.b), cur.bad);
      cur.tiles = tiles_of(cur.length);
      const uint32_t here = (uint32_t)cur.tiles * (uint32_t)a.heads;
      if (rest < here || cur.b + 1 >= a.sequences) break;
      rest -= here;
    }
    cur.h = (int)(rest / (uint32_t)cur.tiles);
    cur.tile = (int)(rest % (uint32_t)cur.tiles);
    fetch_pages(a, cur);

    F32x4 acc[P::kBlocks];
    V8 q[D / 32];
    U32x4 q_next[D / 32];  // the next row's, loading with its first tile
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
    };

    // The loads of a tile, always as many (a tile or half that is not there
    // reads through an empty view): a later wait for one tile then never
    // waits for the next one's.
    const uint32_t ko = (uint32_t)li * a.k_ts + (uint32_t)lg * 16u;
    auto load = [&](const Cursor& c, Tile<D>& t, bool there) -> bool {
      bool bad = c.bad;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int at = c.tile * kTileTokens + 16 * s;
        // rows of the half, those past the sequence's end left out
        const int rows = there ? min(c.length - at, 16) : 0;
        int page = s ? c.page1 : c.page0;
        const bool out = (uint32_t)page >= (uint32_t)a.pages;
        bad |= out && rows > 0;
        page = out ? 0 : page;
        const uint32_t in_page = rows > 0 ? (uint32_t)at & ((1u << a.shift) - 1u) : 0u;
        const bool any = rows > 0 && !out;
        const auto kr = view_of(a.keys + ((int64_t)page * a.k_ps + (int64_t)c.h * a.k_hs) * 2
                                    + (uint64_t)in_page * a.k_ts,
                                any ? (uint32_t)(rows - 1) * a.k_ts + D * 2u : 0u);
        const auto vr = view_of(a.values + ((int64_t)page * a.v_ps + (int64_t)c.h * a.v_hs) * 2
                                    + (uint64_t)in_page * a.v_ts,
                                any ? (uint32_t)(rows - 1) * a.v_ts + D * 2u : 0u);
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
          t.k[s][j] = __builtin_amdgcn_raw_buffer_load_b128(kr, (int)(ko + 64u * j), 0, kStreamLoad);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t vo = (uint32_t)(4 * lg + e) * a.v_ts;
#pragma unroll
          for (int c8 = 0; c8 < P::k8; ++c8)
            t.v8[c8][4 * s + e] = __builtin_amdgcn_raw_buffer_load_b128(
                vr, (int)(vo + li * 16u + 256u * c8), 0, kStreamLoad);
          if constexpr (P::k4 > 0)
            t.v4[4 * s + e] = __builtin_amdgcn_raw_buffer_load_b64(
                vr, (int)(vo + li * 8u + 256u * P::k8), 0, kStreamLoad);
          if constexpr (P::k2 > 0)
            t.v2[4 * s + e] = __builtin_amdgcn_raw_buffer_load_b32(
                vr, (int)(vo + li * 4u + 256u * P::k8 + 128u * P::k4), 0, kTailLoad<D>);
        }
      }
      return bad;
    };

    auto begin_row = [&](const Cursor& c) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j) q[j] = __builtin_bit_cast(V8, q_next[j]);
#pragma unroll
      for (int n = 0; n < P::kBlocks; ++n) acc[n] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m = kNegInf;
      l = 0.0f;
      bad_row = false;
      begun = c.tile == 0;
    };

    // Whether any of the tile's values is infinite or NaN: its product with
    // zeros shows it as NaN.  (8 products more a tile at head_dim 128, on matrix
    // cores that wait for memory: 131072 tokens 91.6 -> 92.1 us, 2003 tokens
    // 11.85 -> 11.94, 128 short sequences at head_dim 64 71.6 -> 72.2.)
    auto has_infinite = [&](const Tile<D>& t) -> bool {
      F32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
      auto add = [&](U32x4 words) { sum = T::mma(__builtin_bit_cast(V8, words), V8{}, sum); };
#pragma unroll
      for (int c8 = 0; c8 < P::k8; ++c8)
#pragma unroll
        for (int e = 0; e < 8; ++e) add(t.v8[c8][e]);
      if constexpr (P::k4 > 0)
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          add(U32x4{t.v4[e][0], t.v4[e][1], t.v4[e + 1][0], t.v4[e + 1][1]});
      if constexpr (P::k2 > 0)
#pragma unroll
        for (int e = 0; e < 8; e += 4) add(U32x4{t.v2[e], t.v2[e + 1], t.v2[e + 2], t.v2[e + 3]});
      return __builtin_amdgcn_ballot_w64(sum[0] + sum[1] + sum[2] + sum[3] != 0.0f) != 0;
    };

    // Ones over the halves of a word that are infinite or NaN (the sum's top
    // bits: exponents of all ones).
    auto infinite_of = [](uint32_t w) -> uint32_t {
      const uint32_t top = (w & 0x7fff7fffu) + (kHalf ? 0x04000400u : 0x00800080u);
      return (top >> 15 & 0x00010001u) * 0xffffu;
    };

    auto compute = [&](const Cursor& c, Tile<D>& t, bool bad, bool last_tile) {
      bad_row |= bad;
      {
        float x[8];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          F32x4 s4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
            s4 = T::mma(__builtin_bit_cast(V8, t.k[s][j]), q[j], s4);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[4 * s + r] = s4[r] * a.scale;
        }
        // rows behind the sequence's end were loaded as zeros and weigh nothing
        const int behind = c.length - c.tile * kTileTokens;
        if (behind < kTileTokens) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = 16 * (e / 4) + 4 * lg + e % 4 < behind ? x[e] : kNegInf;
        }
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, x[e]);
        float u, w;
        xor16_pair(top, u, w);
        top = __builtin_fmaxf(u, w);
        xor32_pair(top, u, w);
        top = __builtin_fmaxf(u, w);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float mn = __builtin_fmaxf(m, top);
          const float by = mn == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= by;
#pragma unroll
          for (int n = 0; n < P::kBlocks; ++n) acc[n] *= by;
        }
        const float base = m == kNegInf ? 0.0f : m;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // (fp16 weights go up to 2^15 instead of 1, and the sum with them, so
          // that those of 2^-24 to 2^-39 of the largest, many in a long
          // context, do not round to zero)
          p[e] = __builtin_amdgcn_exp2f(x[e] - base) * (kHalf ? 32768.0f : 1.0f);
          l += p[e];
        }
        // dims' products: byte permutes gather one dim of two tokens a word
        auto each_product = [&](auto add) {
          constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;
#pragma unroll
          for (int n = 0; n < P::kBlocks; ++n) {
            U32x4 words;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t even, odd;
              int d;
              if (n < 8 * P::k8) {
                d = n % 8;
                even = t.v8[n / 8][2 * e][d / 2];
                odd = t.v8[n / 8][2 * e + 1][d / 2];
              } else if (n < 8 * P::k8 + 4 * P::k4) {
                d = n - 8 * P::k8;
                even = t.v4[2 * e][d / 2];
                odd = t.v4[2 * e + 1][d / 2];
              } else {
                d = n - 8 * P::k8 - 4 * P::k4;
                even = t.v2[2 * e];
                odd = t.v2[2 * e + 1];
              }
              words[e] = __builtin_amdgcn_perm(odd, even, d % 2 ? kHigh : kLow);
            }
            add(n, words);
          }
        };
        if (has_infinite(t)) {
          // Parts of a weight may be 0, and 0 times infinity is NaN: infinities
          // and NaN count here, times 1 (0 where the weight itself is), and as
          // 0 below.
          V8 some;
#pragma unroll
          for (int e = 0; e < 8; ++e) some[e] = (E)(p[e] == 0.0f ? 0.0f : 1.0f);
          each_product([&](int n, U32x4 words) {
#pragma unroll
            for (int e = 0; e < 4; ++e) words[e] &= infinite_of(words[e]);
            acc[n] = T::mma(__builtin_bit_cast(V8, words), some, acc[n]);
          });
#pragma unroll
          for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int c8 = 0; c8 < P::k8; ++c8)
#pragma unroll
              for (int i = 0; i < 4; ++i) t.v8[c8][e][i] &= ~infinite_of(t.v8[c8][e][i]);
            if constexpr (P::k4 > 0)
#pragma unroll
              for (int i = 0; i < 2; ++i) t.v4[e][i] &= ~infinite_of(t.v4[e][i]);
            if constexpr (P::k2 > 0) t.v2[e] &= ~infinite_of(t.v2[e]);
          }
        }
        V8 hi, lo, last;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // the weight as a sum of 16-bit parts that holds all of it: two of
          // fp16 (to 2^-23), three of bf16 (exact).  (Two of bf16 hold it to
          // 2^-17: 1.4 times as many outputs rounded the other way at 131072
          // tokens, and the same 92 us; 128 short sequences at head_dim 64 70.9
          // us against 73.3.)
          hi[e] = (E)p[e];
          const float rest = p[e] - (float)hi[e];
          lo[e] = (E)rest;
          if constexpr (!kHalf) last[e] = (E)(rest - (float)lo[e]);
        }
        auto add_product = [&](int n, U32x4 words) {
          const V8 v = __builtin_bit_cast(V8, words);
          acc[n] = T::mma(v, hi, acc[n]);
          acc[n] = T::mma(v, lo, acc[n]);
          if constexpr (!kHalf) acc[n] = T::mma(v, last, acc[n]);
        };
        each_product(add_product);
      }
      const bool ends = c.tile + 1 == c.tiles;
      if (!ends && !last_tile) return;
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
      Part<D>& part = parts[wave][slot];
      if (lane == 0) heads_s[wave][slot] = PartHead{row, begun, ends, pos - (uint32_t)c.tile,
                                                (uint32_t)c.tiles};
      if (li < a.group) {
        if (lg == 0) part.ml[li] = make_float2(m, sum_l);
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
              *reinterpret_cast<FN*>(&part.acc[li][d + i]) = y;
            }
          });
      }
    };

    Tile<D> t0, t1;
    Cursor ahead = cur, far;  // the tile that is loading, and the one after it
    load_query(cur);
    bool bad0 = load(cur, t0, true), bad1 = false;
    if (left > 1) {
      next_tile(a, ahead);
      fetch_pages(a, ahead);
    }
    bool row_start = true;  // of the row, or of the wave's share of it
    auto step = [&](Tile<D>& now, bool bad, Tile<D>& next) -> bool {
      if (row_start) begin_row(cur);
      if (left > 1 && ahead.tile == 0) load_query(ahead);
      far = ahead;
      if (left > 2) {
        next_tile(a, far);
        fetch_pages(a, far);
      }
      const bool next_bad = load(ahead, next, left > 1);
      compute(cur, now, bad, left == 1);
      cur = ahead;
      ahead = far;
      row_start = cur.tile == 0;
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
      const float2 ml = in ? parts[i / 2][i % 2].ml[g] : make_float2(kNegInf, 0.0f);
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
        const F32x4 p = *reinterpret_cast<const F32x4*>(&parts[i / 2][i % 2].acc[g][d]);
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
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedArgs a) {
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

PagedPlan paged_plan(const rkv_paged_cache* c, int64_t group) {
  PagedPlan P;
  RKV_DISPATCH_DIM(c->dim, D, P.grid = compute_units() * kPerCu<D>);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t parts = (size_t)P.grid * 2;
  P.ml_off = up(P.grid * kOpenStride * sizeof(int2));
  P.acc_off = P.ml_off + up(parts * group * sizeof(float2));
  P.total = P.acc_off + up(parts * group * c->dim * sizeof(float));
  return P;
}

int check_paged(const char* who, const rkv_paged_cache* c, int64_t group) {
  int rc = check_cache(who, c);
  if (rc) return rc;
  if (c->dtype != RKV_BF16 && c->dtype != RKV_F16)
    return set_error(kUnsupported, "%s: the cache must be bfloat16 or float16", who);
  if (!supported_dim(c->dim))
    return set_error(kUnsupported, "%s: head_dim %lld not in 32..256 step 32", who,
                     (long long)c->dim);
  if (group <= 0) return set_error(kInvalidArgument, "%s: empty group", who);
  if (group > kMaxGroup)
    return set_error(kUnsupported, "%s: GQA group %lld exceeds 16", who, (long long)group);
  const int64_t strides[] = {
      read_stride(c->key_page_stride, c->pages),   read_stride(c->key_head_stride, c->heads),
      read_stride(c->value_page_stride, c->pages), read_stride(c->value_head_stride, c->heads),
      c->key_token_stride,                         c->value_token_stride};
  for (int64_t s : strides)
    if (s % 8) return set_error(kInvalidArgument, "%s: cache strides must be multiples of 8", who);
  if (c->key_token_stride < c->dim || c->value_token_stride < c->dim)
    return set_error(kInvalidArgument, "%s: row strides must be >= head_dim", who);
  // tiles and rows are counted in 32 bits
  const int64_t tiles = c->max_blocks * c->page_size / kTileTokens + 1;
  if (tiles > ((int64_t(1) << 31) - 1) / c->heads / c->sequences)
    return set_error(kUnsupported, "%s: the block table covers too many tokens", who);
  // 16 rows of a page are addressed with 32-bit byte offsets
  if (c->key_token_stride > (1 << 25) || c->value_token_stride > (1 << 25))
    return set_error(kUnsupported, "%s: rows more than 64 MiB apart", who);
  if (!aligned(c->keys, 16) || !aligned(c->values, 16))
    return set_error(kInvalidArgument, "%s: the cache must be 16-byte aligned", who);
  return kOk;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_paged_plan(const rkv_paged_cache* cache, int64_t group,
                              size_t* workspace_bytes) {
  clear_error();
  if (!workspace_bytes) return set_error(kInvalidArgument, "rkv_paged_plan: null pointer");
  const int rc = check_paged("rkv_paged_plan", cache, group);
  if (rc) return rc;
  *workspace_bytes = paged_plan(cache, group).total;
  return kOk;
}

extern "C" int rkv_paged_decode(const rkv_paged_cache* cache, const void* query,
                                int64_t q_sequence_stride, int64_t q_head_stride, int64_t group,
                                float scale, void* output, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  const char* who = "rkv_paged_decode";
  clear_error();
  const int rc = check_paged(who, cache, group);
  if (rc) return rc;
  if (!query || !output) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  q_sequence_stride = read_stride(q_sequence_stride, cache->sequences);
  q_head_stride = read_stride(q_head_stride, cache->heads * group);
  if (q_sequence_stride < 0 || q_head_stride < 0 || q_head_stride > (1 << 25))
    return set_error(kUnsupported, "%s: query stride", who);
  if (!aligned(query, 16) || !aligned(output, 16) || q_sequence_stride % 8 || q_head_stride % 8)
    return set_error(kInvalidArgument,
                     "%s: query and output must be 16-byte aligned with strides in multiples of 8",
                     who);
  if (rows_meet_pages(cache, output, cache->heads * group * cache->dim, cache->dim,
                      cache->sequences, cache->heads * group))
    return set_error(kInvalidArgument, "%s: output overlaps the cache", who);
  const PagedPlan P = paged_plan(cache, group);
  if (!workspace || workspace_bytes < P.total)
    return set_error(kWorkspaceTooSmall, "%s: workspace of %zu bytes, %zu needed", who,
                     workspace_bytes, P.total);
  if (!aligned(workspace, 16))
    return set_error(kInvalidArgument, "%s: workspace must be 16-byte aligned", who);
  PagedArgs a{};
  a.query = static_cast<const char*>(query);
  a.q_bs = q_sequence_stride;
  a.q_hs = q_head_stride;
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.k_ps = read_stride(cache->key_page_stride, cache->pages);
  a.k_hs = read_stride(cache->key_head_stride, cache->heads);
  a.v_ps = read_stride(cache->value_page_stride, cache->pages);
  a.v_hs = read_stride(cache->value_head_stride, cache->heads);
  a.k_ts = (uint32_t)(cache->key_token_stride * 2);
  a.v_ts = (uint32_t)(cache->value_token_stride * 2);
  a.table = cache->block_table;
  a.table_stride = cache->table_stride;
  a.lengths = cache->lengths;
  a.sequences = (int)cache->sequences;
  a.heads = (int)cache->heads;
  a.group = (int)group;
  a.max_blocks = (int)cache->max_blocks;
  a.pages = (int)cache->pages;
  a.shift = page_shift(cache->page_size);
  a.scale = scale * kLog2e;
  a.out = static_cast<char*>(output);
  char* ws = static_cast<char*>(workspace);
  a.open = reinterpret_cast<int2*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + P.ml_off);
  a.part_acc = reinterpret_cast<float*>(ws + P.acc_off);
  const dim3 join((unsigned)P.grid, (unsigned)group);
  RKV_DISPATCH_DIM(cache->dim, D, {
    if (cache->dtype == RKV_F16) {
      paged_kernel<D, true><<<dim3(P.grid), dim3(kThreads), 0, stream>>>(a);
      paged_join_kernel<D, true><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    } else {
      paged_kernel<D, false><<<dim3(P.grid), dim3(kThreads), 0, stream>>>(a);
      paged_join_kernel<D, false><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    }
  });
  return check_launch("paged_kernel");
}
