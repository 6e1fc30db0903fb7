// Attention of prompts' rows, over rows of their own sequences
// (rkv_prompt_attention) or over a paged cache (rkv_paged_prompt):
//   out[i, h] = softmax_j(f(scale q[i, h] . K[j])) V
// over the tokens j of i's sequence that i sees: those up to i, and those of
// the sequence's prefix, at most `window` back; f caps the scores and biases
// them by distance.
#include <algorithm>

#include "rkv_paged_walk.h"

namespace rkv {
namespace {

constexpr int kPromptThreads = 256;
constexpr int kWaveRows = 32;                     // query rows of a wave
constexpr int kTileRows = 4 * kWaveRows;          // of a workgroup

typedef short S16x4 __attribute__((ext_vector_type(4)));
typedef float F32x16 __attribute__((ext_vector_type(16)));

template <bool kHalf>
__device__ __forceinline__ F32x16 mma32(const U32x4& a, const U32x4& b, F32x16 c) {
  if constexpr (kHalf)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(typename Type16<true>::V8, a),
        __builtin_bit_cast(typename Type16<true>::V8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(typename Type16<false>::V8, a),
        __builtin_bit_cast(typename Type16<false>::V8, b), c, 0, 0, 0);
}

struct PromptArgs {
  const char* query;           // (tokens, H G, D)
  int64_t q_ts, q_hs;          // token and head strides, elements
  const char* keys;            // rows (key tokens, H, D), or a cache's pages
  const char* values;
  int64_t k_ps, k_hs, v_ps, v_hs;  // page (rows: none) and head strides, elements
  uint32_t k_ts, v_ts;         // row strides, bytes
  const int32_t* starts;       // [sequences + 1] of the query rows (null: one sequence)
  const int32_t* key_starts;   // of the key rows (null: as starts)
  const int32_t* lengths;      // paged: the sequences' tokens
  const int32_t* table;        // paged (null: rows)
  int64_t table_stride;
  const int32_t* prefix;       // [sequences] tokens that all rows see (null: none)
  int sequences, heads, group, max_blocks, pages, shift;
  int tokens, key_tokens;
  int step;                    // starts are implied: sequence b has row b alone
  float scale;                 // magnitude, times log2 e
  uint32_t flip;               // on the query's words: the scale's sign
  float cap, per_cap;          // as WalkArgs
  const float* slopes;
  int window;
  char* out;                   // (tokens, H G, D) dense
  int zero_rest;               // workgroups a head for the rows of no sequence, which
                               // become zeros (0: they stay as they were)
  int tiles;                   // at most so many in the grid
  // few tiles: so many workgroups share all tiles' keys (0: each has a tile of
  // its own); keys are counted in units of 2^unit LDS tiles
  int shares, unit;
  float2* part_ml;             // [workgroup][kTileRows]
  float* part_acc;             // [..][D]
};

// Keys of a tile in LDS: 64, 32 at head dims whose accumulators take the
// registers of two waves.
template <int D>
struct PromptTile {
  static constexpr int kTokens = D <= 128 ? 64 : 32;
  // Rows 16 bytes more than a multiple of 32 apart: 16 lanes that read one
  // column of 16 rows take all banks.
  static constexpr int kKeyRow = 2 * D + 16;
  // An odd multiple of 64 bytes: 4 rows of 64 bytes, as a transposing read of
  // half a wave takes them, lie in different banks.
  static constexpr int kValueRow = 2 * D + (D / 32 % 2 ? 0 : 64);
  static constexpr int kValueAt = kTokens * kKeyRow;
  static constexpr int kBytes = kValueAt + kTokens * kValueRow;
};

// A sequence's query rows, and where the workgroup's tile stands in them.
struct PromptRows {
  int b, first, count;  // sequence, its first row, its rows
  int tile;             // of kTileRows (row, head of the group) pairs
};

// Sequence b's rows, inside the tensor.  False: its starts decrease.
__device__ __forceinline__ bool rows_of(const PromptArgs& a, int b, int& first, int& count) {
  int from, to;
  if (a.step) {
    from = b;
    to = b + 1;
  } else if (a.starts) {
    from = a.starts[b];
    to = a.starts[b + 1];
  } else {
    from = 0;
    to = a.tokens;
  }
  first = min(max(from, 0), a.tokens);
  count = min(max(to, first), a.tokens) - first;
  return from <= to;
}

__device__ __forceinline__ uint32_t tiles_for(const PromptArgs& a, int count) {
  return (uint32_t)(((int64_t)count * a.group + kTileRows - 1) / kTileRows);
}

// A sequence's keys: their number (0, and `bad`, for a length past its table)
// and, of rows, the first one.
__device__ __forceinline__ int keys_of(const PromptArgs& a, const PromptRows& r, int& first,
                                       bool& bad) {
  first = 0;
  bad = false;
  if (a.table) {
    const int n = a.lengths[r.b];
    bad = n > 0 && (n - 1) >> a.shift >= a.max_blocks;
    return bad || n < 0 ? 0 : n;
  }
  if (a.key_starts) {
    first = min(max(a.key_starts[r.b], 0), a.key_tokens);
    return min(max(a.key_starts[r.b + 1], first), a.key_tokens) - first;
  }
  first = r.first;
  return r.count;
}

// The slot-th of the entries that the sequences have `entries(b, odd)` of, with its
// sequence and its place among that one's entries.  False: there are fewer, or a
// sequence's starts decrease (odd): overlapping sequences could have more entries
// than the grid, so that then no row is any sequence's.
template <typename Entries>
__device__ __forceinline__ bool find_entry(const PromptArgs& a, uint32_t slot, bool from_end,
                                           Entries entries, int& b, uint32_t& place) {
  const int lane = threadIdx.x % kWave;
  const int per = (a.sequences + kWave - 1) / kWave;
  uint32_t sum = 0;
  bool odd = false;
  for (int i = 0; i < per && lane * per + i < a.sequences; ++i) sum += entries(lane * per + i, odd);
  const uint32_t upto = wave_scan(sum);
  const uint32_t total = (uint32_t)uniform((int)__shfl((int)upto, kWave - 1, kWave));
  if (slot >= total || __builtin_amdgcn_ballot_w64(odd) != 0) return false;
  const uint32_t at = from_end ? total - 1u - slot : slot;
  const int owner = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > at));
  place = at - (uint32_t)uniform(__shfl((int)(upto - sum), owner, kWave));
  for (b = owner * per; b < a.sequences; ++b) {
    const uint32_t here = (uint32_t)uniform((int)entries(b, odd));
    if (place < here) return true;
    place -= here;
  }
  return false;  // (starts that change under the call)
}

// The slot-th of the tiles, the last ones of the last sequence first: a
// sequence's later tiles have more keys.
__device__ __forceinline__ bool find_tile(const PromptArgs& a, uint32_t slot, PromptRows& r) {
  uint32_t place;
  auto tiles = [&](int b, bool& odd) {
    int first, count;
    odd |= !rows_of(a, b, first, count);
    return tiles_for(a, count);
  };
  if (!find_entry(a, slot, true, tiles, r.b, place)) return false;
  rows_of(a, r.b, r.first, r.count);
  r.first = uniform(r.first);
  r.count = uniform(r.count);
  r.tile = (int)place;
  return true;
}

// A tile's part of its sequence's keys, for one head.
struct Share {
  int head, chunk, chunks;  // of the sequence's keys
  int begin, end;           // LDS tiles of the chunk
  int first, apart;         // the tile's first chunk among all shares, and from one to the next
};

// The sequence's range of LDS tiles with keys that its rows see, in units.
template <int T>
__device__ __forceinline__ uint32_t units_of(const PromptArgs& a, const PromptRows& r,
                                             int& begin) {
  int first;
  bool bad;
  const int length = keys_of(a, r, first, bad), at = max(length - r.count, 0);
  begin = at >= a.window ? (at - a.window + 1) / T : 0;
  const int tiles = (int)(((int64_t)length + T - 1) / T) - begin;
  return tiles > 0 ? (uint32_t)(((int64_t)tiles + (1 << a.unit) - 1) >> a.unit) : 1u;
}

// Shares of few tiles' keys: chunks of so many units that all fit the grid
// (rounding up costs a tile one chunk at most), 256 keys at least.  They lie
// sequence by sequence, chunk by chunk, head by head, tile by tile: a chunk's
// tiles are neighbours.  The slot-th of them, or (kJoin) the first of the slot-th
// tile and head.
template <int T, bool kJoin>
__device__ __forceinline__ bool find_share(const PromptArgs& a, uint32_t slot, PromptRows& r,
                                           Share& share) {
  const int lane = threadIdx.x % kWave;
  const int per = (a.sequences + kWave - 1) / kWave;
  auto sizes = [&](int b, uint32_t& tiles, uint32_t& units, int& begin) {
    PromptRows q;
    q.b = b;
    const bool odd = !rows_of(a, b, q.first, q.count);
    tiles = tiles_for(a, q.count);
    units = tiles ? units_of<T>(a, q, begin) : 0u;
    return odd;
  };
  uint32_t sum = 0, tiles, units;
  int begin = 0;
  for (int i = 0; i < per && lane * per + i < a.sequences; ++i) {
    sizes(lane * per + i, tiles, units, begin);
    sum += tiles * units;
  }
  const uint32_t all = (uint32_t)uniform(
      (int)__shfl((int)wave_scan(sum), kWave - 1, kWave));
  const uint32_t heads = (uint32_t)a.heads, room = (uint32_t)a.shares - (uint32_t)a.tiles * heads;
  const uint64_t need = ((uint64_t)all * heads + room - 1u) / room;
  const uint32_t least = max(256 / T >> a.unit, 1);
  const uint32_t chunk = need > least ? (uint32_t)need : least;
  auto chunks_of = [&](uint32_t n) { return (n + chunk - 1u) / chunk; };
  auto entries = [&](int b, bool& odd) {
    odd |= sizes(b, tiles, units, begin);
    return tiles * heads * (kJoin ? 1u : chunks_of(units));
  };
  uint32_t place;
  if (!find_entry(a, slot, false, entries, r.b, place)) return false;
  rows_of(a, r.b, r.first, r.count);
  r.first = uniform(r.first);
  r.count = uniform(r.count);
  tiles = tiles_for(a, r.count);
  units = (uint32_t)uniform((int)units_of<T>(a, r, begin));
  r.tile = (int)(place % tiles);
  share.head = (int)(place / tiles % heads);
  share.chunk = (int)(place / tiles / heads);
  share.chunks = (int)chunks_of(units);
  share.apart = (int)(tiles * heads);
  const int64_t from = ((int64_t)share.chunk * chunk << a.unit) + uniform(begin);
  share.begin = (int)min(from, (int64_t)INT32_MAX);
  share.end = (int)min(from + ((int64_t)chunk << a.unit), (int64_t)INT32_MAX);
  if constexpr (kJoin) {
    uint32_t before = 0;  // shares of the sequences before
    for (int i = 0; i < per && lane * per + i < r.b; ++i) {
      sizes(lane * per + i, tiles, units, begin);
      before += tiles * heads * chunks_of(units);
    }
    share.first = uniform(__shfl((int)wave_scan(before), kWave - 1, kWave)) + (int)place;
  }
  return true;
}

// Rows of no sequence (all, where starts decrease): the part-th part of them becomes
// zeros, for one head's group.
template <int D>
__device__ __forceinline__ void zero_rows(const PromptArgs& a, int head, int part) {
  int first, count, last;
  bool odd = false;
  for (int b = (int)threadIdx.x % kWave; b < a.sequences; b += kWave)
    odd |= !rows_of(a, b, first, count);
  rows_of(a, 0, first, count);
  rows_of(a, a.sequences - 1, last, count);
  last += count;
  if (__builtin_amdgcn_ballot_w64(odd) != 0) last = first;
  const int per_row = a.group * (D / 8);
  const int64_t n = (int64_t)(a.tokens - last + first) * per_row;
  for (int64_t i = (int64_t)part * kPromptThreads + threadIdx.x; i < n;
       i += (int64_t)a.zero_rest * kPromptThreads) {
    const int64_t row = i / per_row, token = row < first ? row : row - first + last;
    reinterpret_cast<U32x4*>(a.out)[(token * a.heads + head) * per_row + i % per_row] =
        U32x4{0u, 0u, 0u, 0u};
  }
}

// What a row's sums are multiplied with: 0 for one that sees nothing, NaN for one
// whose scores are -inf alone or NaN.
__device__ __forceinline__ float weight_of(bool sees, float l) {
  return !sees ? 0.0f : l > 0.0f ? 1.0f / l : __builtin_nanf("");
}

// An infinite or NaN value makes NaN of every row whose products it is in, those
// that do not see it as well.  A workgroup that ends with such rows goes over
// its keys again: once for the outputs that see +inf or NaN, once for those that
// see -inf or NaN, each with ones for such values and for the weights of keys
// that are seen; then with zeros for all of them.
enum Pass : int { kPlain, kUp, kDown, kFinite };

// What a word of two values is in a pass.
template <bool kHalf>
__device__ __forceinline__ uint32_t value_words(uint32_t w, int pass) {
  constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u, kOne = kHalf ? 0x3c00u : 0x3f80u;
  uint32_t to = 0;
#pragma unroll
  for (int k = 0; k < 32; k += 16) {
    const uint32_t v = w >> k & 0xffffu;
    const bool odd = (v & kExp) == kExp, nan = (v & 0x7fffu) > kExp;
    const bool counts = odd && (nan || (v >> 15 != 0u) == (pass == kDown));
    to |= (pass == kFinite ? (odd ? 0u : v) : counts ? kOne : 0u) << k;
  }
  return to;
}

// The matrix cores and the softmax's vector issue bound it, one after the other
// more than side by side: 16384 tokens (8 KV heads, group 4, d 128) in 2170-2240
// us, 980-1010 TFLOP/s of the visible products (a bf16 product of 8192^3 reaches 1257
// here), the matrix cores busy for 47 % of it and the vector ALUs for 51 %.
// (Scores of the next tile computed beside the softmax of this one, keys two tiles
// ahead: 2610 us; tiles of 32 keys 2380; reads of all a product's operands in
// groups of 8: 2300 against 2255.)  Few rows over many keys are bound by the keys
// on their way into LDS: 3 x 33 rows over 134 K tokens of 4 heads (274 MB) 104-120
// us, then 12 for the join.  One tile alone takes 10 us: finding it, its first
// loads and its code.
// A workgroup has 128 (row, head of the group) pairs of one sequence and KV
// head, 32 a wave, and goes over the keys they see in tiles that two LDS buffers
// hold: the next one's rows are on their way to registers while one is computed.
// As in the decode the query rows are the products' columns, so that a lane's
// maximum, sum and accumulators belong to one of them (lanes l and l + 32
// share row l % 32):
//   S^T = K Q^T: A = 32 keys (lane l: key l % 32, dims 16 j + 8 (l / 32) ..),
//     B = the query rows; lane l gets the keys 8 (i / 4) + 4 (l / 32) + i % 4,
//     i = 0..15.
//   O^T = V^T P^T: B = 16 keys' weights as the lane has them, slot e of 8: key
//     8 (e / 4) + 4 (l / 32) + e % 4.  A = V^T over the same slots: two
//     transposing reads of 4 keys x 16 dims.
template <int D, bool kHalf, bool kScores>
__global__ __launch_bounds__(kPromptThreads)
__attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void prompt_kernel(PromptArgs a) {
  using Tile = PromptTile<D>;
  using E = typename Type16<kHalf>::E;
  constexpr int T = Tile::kTokens, kGroups = T / 16, kLoads = D / 32;
  constexpr int kOwn = T == 64 ? 2 : 1;  // tensors of which a wave loads 16 rows a tile
  constexpr int kMarks = (D / 32 + 1) / 2;
  // Of the two waves of a SIMD the one in its products goes first, so that the
  // other's softmax runs beside them (16384 tokens, head_dim 128, 2300 -> 2180 us);
  // where the softmax takes longer it goes first (head_dim 64, 8192 tokens of 16
  // heads, 218 -> 204 us).
  constexpr bool kProductsFirst = D > 64;
  __shared__ alignas(16) char smem[2][Tile::kBytes];
  __shared__ uint32_t marks[2][kMarks][kPromptThreads];  // outputs that kUp and kDown found
  const uint32_t last = gridDim.x - (uint32_t)(a.zero_rest * a.heads);
  if (blockIdx.x >= last) {
    const int rest = (int)(blockIdx.x - last);
    zero_rows<D>(a, rest % a.heads, rest / a.heads);
    return;
  }
  PromptRows rows;
  Share share{(int)(blockIdx.x % (uint32_t)a.heads), 0, 1, 0, INT32_MAX, 0, 0};
  // A chunk's tiles go to one XCD (workgroups go to the 8 in turn), whose L2 then
  // has the keys of the second from the first.
  const uint32_t each = (uint32_t)a.shares / 8u;
  const uint32_t slot = blockIdx.x < each * 8u ? blockIdx.x % 8u * each + blockIdx.x / 8u
                                               : blockIdx.x;
  if (!(a.shares ? find_share<T, false>(a, slot, rows, share)
                 : find_tile(a, blockIdx.x / (uint32_t)a.heads, rows)))
    return;
  const int head = share.head;
  const int lane = threadIdx.x % kWave, wave = uniform((int)threadIdx.x / kWave);
  const int l32 = lane & 31, h = lane >> 5;

  // ---- the sequence's keys
  int key_first;
  bool bad;
  int length = keys_of(a, rows, key_first, bad);
  length = uniform(length);
  key_first = uniform(key_first);
  bad = uniform(bad);
  int prefix = a.prefix ? scalar_at(a.prefix, rows.b) : 0;
  prefix = min(max(prefix, 0), length);

  // ---- this lane's row, and the keys that the workgroup and the wave see
  const int pairs = rows.count * a.group;
  const int base_pos = length - rows.count;
  auto position_of = [&](int pair) { return base_pos + pair / a.group; };
  const int pair0 = rows.tile * kTileRows, pair = pair0 + wave * kWaveRows + l32;
  const bool mine = pair < pairs;
  const int in_seq = mine ? pair / a.group : 0, g = mine ? pair % a.group : 0;
  const int pos = base_pos + in_seq;
  // keys low < j <= lim are seen
  const bool sees = mine && pos >= 0;
  const int lim = sees ? max(pos, prefix - 1) : -1;
  const int low = sees ? (pos >= a.window ? pos - a.window : -1) : -1;
  auto range = [&](int from, int to, int& begin, int& end) {  // of pairs from .. to - 1
    const int p0 = max(position_of(from), 0), p1 = position_of(min(to, pairs) - 1);
    begin = p0 >= a.window ? p0 - a.window + 1 : 0;
    end = from >= pairs || p1 < 0 ? 0 : min(max(p1 + 1, prefix), length);
  };
  int wg_begin, wg_end, wave_begin, wave_end;
  range(pair0, pair0 + kTileRows, wg_begin, wg_end);
  range(pair0 + wave * kWaveRows, pair0 + (wave + 1) * kWaveRows, wave_begin, wave_end);
  // keys that every row of the wave sees: whole_begin .. whole_end - 1
  int whole_begin, whole_end;
  {
    const int from = pair0 + wave * kWaveRows, to = min(from + kWaveRows, pairs) - 1;
    const int p0 = position_of(from), p1 = position_of(max(to, from));
    whole_end = p0 < 0 ? 0 : max(p0 + 1, prefix);
    whole_begin = p1 >= a.window ? p1 - a.window + 1 : 0;
  }
  const int tile_begin = max(wg_begin / T, share.begin);
  const int tile_end = min((int)(((int64_t)wg_end + T - 1) / T), share.end);

  // ---- the query rows
  U32x4 q[D / 16];
  {
    const char* from = a.query + ((int64_t)(rows.first + in_seq) * a.q_ts +
                                  (int64_t)(head * a.group + g) * a.q_hs) * 2 + h * 16;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      q[j] = mine ? *reinterpret_cast<const U32x4*>(from + 32 * j) : U32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 4; ++i) q[j][i] ^= a.flip;
    }
  }
  // Scores without a cap are scaled on the way into the exponential, slopes divided
  // by the scale for it; of tiles before all the wave's rows a key's bias is that of
  // the tile's first and its place's, one operation a score (23 documents, head_dim
  // 64, 119 -> 111 us then, 108 now).  Not with slopes or scales whose products could overflow.
  float slope = 0.0f, unit_slope = 0.0f, scale = a.scale;
  bool late = true;
  int biased_end = 0;  // tokens up to every row of the wave
  if constexpr (kScores) {
    if (a.slopes) slope = a.slopes[head * a.group + g] * kLog2e;
    const bool tame = __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(slope) < 1e20f)) == 0;
    late = tame && !(a.cap > 0.0f) && a.scale > 0x1p-20f && a.scale < 0x1p20f;
    unit_slope = late ? slope / a.scale : slope;
    scale = late ? a.scale : 1.0f;
    if (tame) biased_end = position_of(pair0 + wave * kWaveRows) + 1;
  }

  int pass = kPlain;

  // ---- a wave's 16 rows of a tile: of keys and values, or (32 tokens) of one
  const int group16 = wave % kGroups;
  const bool of_values = kOwn == 1 && wave >= 2;
  U32x4 staged[kOwn][kLoads];
  bool staged_bad = false;
  const int64_t block_row = (int64_t)rows.b * a.table_stride;
  auto page_of = [&](int tile) {
    const int at = tile * T + 16 * group16;
    return a.table ? scalar_at(a.table, block_row + (at < length ? at >> a.shift : 0)) : 0;
  };
  // (row, byte) of the lane's i-th 16 bytes of a unit
  auto unit_row = [&](int i) { return (i * kWave + lane) / (D / 8); };
  auto unit_byte = [&](int i) { return (i * kWave + lane) % (D / 8) * 16; };
  auto load = [&](int tile, int page) {
    const int at = tile * T + 16 * group16;
    const int n = min(length - at, 16);
    const bool out = a.table && (uint32_t)page >= (uint32_t)a.pages;
    staged_bad = out && n > 0;
    const bool any = n > 0 && !out;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const bool values = kOwn == 2 ? k == 1 : of_values;
      const uint32_t ts = values ? a.v_ts : a.k_ts;
      const int64_t hs = values ? a.v_hs : a.k_hs, ps = values ? a.v_ps : a.k_ps;
      const char* base = (values ? a.values : a.keys) + (int64_t)head * hs * 2;
      if (a.table)
        base += (any ? (int64_t)page * ps * 2 : 0) +
                (int64_t)(any ? at & ((1 << a.shift) - 1) : 0) * ts;
      else
        base += (int64_t)(any ? key_first + at : 0) * ts;
      const auto view = view_of(base, any ? (uint32_t)(n - 1) * ts + D * 2u : 0u);
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        staged[k][i] = __builtin_amdgcn_raw_buffer_load_b128(
            view, (int)((uint32_t)unit_row(i) * ts + (uint32_t)unit_byte(i)), 0, 0);
    }
  };
  auto store = [&](char* buffer) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const bool values = kOwn == 2 ? k == 1 : of_values;
      if (staged_bad && !values) {
        // (keys of a page that is not there: whoever sees them gets NaN)
        constexpr uint32_t kNan = kHalf ? 0x7e007e00u : 0x7fc07fc0u;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) staged[k][i] = U32x4{kNan, kNan, kNan, kNan};
      }
      if (pass != kPlain && values) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) staged[k][i][j] = value_words<kHalf>(staged[k][i][j], pass);
      }
      char* to = buffer + (values ? Tile::kValueAt : 0);
      const int stride = values ? Tile::kValueRow : Tile::kKeyRow;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *reinterpret_cast<U32x4*>(to + (16 * group16 + unit_row(i)) * stride + unit_byte(i)) =
            staged[k][i];
    }
  };

  F32x16 acc[D / 32];
  float m, l;
  for (;;) {
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][i] = 0.0f;
    m = kNegInf;
    l = 0.0f;
    int page_next = 0;
    if (tile_begin < tile_end) {
      load(tile_begin, page_of(tile_begin));
      page_next = page_of(tile_begin + 1);
      store(smem[0]);
    }
    __syncthreads();
    for (int tile = tile_begin; tile < tile_end; ++tile) {
      const char* buffer = smem[(tile - tile_begin) & 1];
      const bool more = tile + 1 < tile_end;
      if (more) {
        load(tile + 1, page_next);
        page_next = page_of(tile + 2);
      }
      const int t0 = tile * T;
      if (t0 < wave_end && t0 + T > wave_begin) {
        __builtin_amdgcn_s_setprio(kProductsFirst ? 1 : 0);
        // ---- scores
        F32x16 s[T / 32];
#pragma unroll
        for (int u = 0; u < T / 32; ++u) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
          const char* keys = buffer + (32 * u + l32) * Tile::kKeyRow + 16 * h;
          // (4 reads ahead of the products)
          constexpr int kAhead = 4;
          U32x4 k[D / 16];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) k[j] = *reinterpret_cast<const U32x4*>(keys + 32 * j);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) s[u] = mma32<kHalf>(k[j], q[j], s[u]);
          __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (j + kAhead < D / 16) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
        }
        __builtin_amdgcn_s_setprio(kProductsFirst ? 0 : 1);
        auto token = [&](int u, int i) { return t0 + 32 * u + 8 * (i / 4) + 4 * h + i % 4; };
        float bias = 0.0f;  // of the lane's first key, apart from the scores
        if constexpr (kScores) {
          const float by = a.cap > 0.0f ? a.per_cap : a.scale;
          if (!late) {
#pragma unroll
            for (int u = 0; u < T / 32; ++u) s[u] *= by;
          }
          if (a.cap > 0.0f) {
#pragma unroll
            for (int u = 0; u < T / 32; ++u)
#pragma unroll
              for (int i = 0; i < 16; ++i) s[u][i] = tanh_hw(s[u][i]) * a.cap;
          }
          if (a.slopes) {
            // the distance of a lane's first key, and its others' from that
            const float far = (float)(pos - token(0, 0));
            if (t0 + T <= biased_end) {
              bias = -slope * far;
#pragma unroll
              for (int u = 0; u < T / 32; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  s[u][i] = __builtin_fmaf(unit_slope, (float)(32 * u + 8 * (i / 4) + i % 4),
                                           s[u][i]);
            } else {
#pragma unroll
              for (int u = 0; u < T / 32; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  s[u][i] = __builtin_fmaf(
                      -unit_slope, __builtin_fabsf(far - (float)(32 * u + 8 * (i / 4) + i % 4)),
                      s[u][i]);
            }
          }
        }
        if (t0 + T > whole_end || t0 < whole_begin) {
#pragma unroll
          for (int u = 0; u < T / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              s[u][i] = token(u, i) <= lim && token(u, i) > low ? s[u][i] : kNegInf;
        }
        // ---- weights
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < T / 32; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[u][i]);
        top = kScores ? __builtin_fmaf(top, scale, bias) : top * scale;
        float x, y;
        xor32_pair(top, x, y);
        top = __builtin_fmaxf(x, y);
        // (the maximum may lag by 2^8: weights up to that, and fewer rescalings)
        if (__builtin_amdgcn_ballot_w64(top > m + 8.0f) != 0) {
          const float mn = __builtin_fmaxf(m, top);
          // (kUp and kDown count: a count does not shrink)
          const float by = mn == kNegInf || pass == kUp || pass == kDown
                               ? 1.0f
                               : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= by;
#pragma unroll
          for (int n = 0; n < D / 32; ++n) acc[n] *= by;
        }
        // (fp16 weights start from 2^7: those under 2^-24 of the largest, many
        // in a long context, do not all round to zero)
        const float base = (m == kNegInf ? 0.0f : kHalf ? m - 7.0f : m) - bias;
        U32x4 p[T / 16];
#pragma unroll
        for (int u = 0; u < T / 32; ++u)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            typedef E E2 __attribute__((ext_vector_type(2)));
            const float p0 =
                __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], scale, -base));
            const float p1 =
                __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i + 1], scale, -base));
            l += p0;
            l += p1;
            // A weight is rounded to 16 bits, as the products take it: 2^-9 of it in
            // bf16, half of what an output's own rounding may be off by.
            p[2 * u + i / 8][i % 8 / 2] = __builtin_bit_cast(uint32_t, E2{(E)p0, (E)p1});
          }
        if (pass == kUp || pass == kDown) {  // every key that is seen counts once
#pragma unroll
          for (int u = 0; u < T / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              constexpr uint32_t kOne = kHalf ? 0x3c00u : 0x3f80u;
              auto seen = [&](int e) { return token(u, e) <= lim && token(u, e) > low; };
              p[2 * u + i / 8][i % 8 / 2] = (seen(i) ? kOne : 0u) | (seen(i + 1) ? kOne << 16 : 0u);
            }
        }
        __builtin_amdgcn_s_setprio(kProductsFirst ? 1 : 0);
        // ---- products
        const int l16 = lane & 15;
        const char* values = buffer + Tile::kValueAt + (4 * h + l16 / 4) * Tile::kValueRow +
                             32 * (lane >> 4 & 1) + 8 * (l16 % 4);
#pragma unroll
        for (int c = 0; c < T / 16; ++c)
#pragma unroll
          for (int n = 0; n < D / 32; ++n) {
            U32x4 v;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              typedef __attribute__((address_space(3))) S16x4 Lds;
              const auto w = __builtin_bit_cast(
                  U32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                             (Lds*)(values + (16 * c + 8 * k) * Tile::kValueRow + 64 * n)));
              v[2 * k] = w[0];
              v[2 * k + 1] = w[1];
            }
            acc[n] = mma32<kHalf>(v, p[c], acc[n]);
          }
        __builtin_amdgcn_s_setprio(0);
      }
      if (more) store(smem[(tile + 1 - tile_begin) & 1]);
      __syncthreads();
    }
    if (pass == kFinite) break;
    if (pass == kPlain) {
      float sum = 0.0f;  // finite values times 0: NaN if one is not
#pragma unroll
      for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = __builtin_fmaf(acc[n][i], 0.0f, sum);
      if (!__syncthreads_or(sum != 0.0f)) break;
      pass = kUp;
      continue;
    }
#pragma unroll
    for (int w = 0; w < kMarks; ++w) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (2 * w + i / 16 < D / 32) bits |= acc[2 * w + i / 16][i % 16] != 0.0f ? 1u << i : 0u;
      marks[pass - kUp][w][threadIdx.x] = bits;
    }
    pass = pass == kUp ? kDown : kFinite;
  }
  if (pass == kFinite) {
#pragma unroll
    for (int n = 0; n < D / 32; ++n) {
      const uint32_t up = marks[0][n / 2][threadIdx.x] >> (16 * (n % 2));
      const uint32_t down = marks[1][n / 2][threadIdx.x] >> (16 * (n % 2));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool u = up >> i & 1u, d = down >> i & 1u;
        acc[n][i] += u && d ? __builtin_nanf("") : u ? kPosInf : d ? kNegInf : 0.0f;
      }
    }
  }

  // ---- the rows
  float x, y;
  xor32_pair(l, x, y);
  l = x + y;
  if (!mine) return;
  if (bad) l = __builtin_nanf("");
  const int64_t row = (int64_t)(rows.first + in_seq) * (a.heads * a.group) + head * a.group + g;
  if (share.chunks > 1) {
    const int64_t at = (int64_t)slot * kTileRows + (pair - pair0);
    float* to = a.part_acc + at * D + 4 * h;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<F32x4*>(to + 32 * n + 8 * k) =
            F32x4{acc[n][4 * k], acc[n][4 * k + 1], acc[n][4 * k + 2], acc[n][4 * k + 3]};
    if (h == 0) a.part_ml[at] = make_float2(m, l);
    return;
  }
  const float by = weight_of(sees || bad, l);
  char* to = a.out + row * (D * 2) + 8 * h;
#pragma unroll
  for (int n = 0; n < D / 32; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      typedef E E4 __attribute__((ext_vector_type(4)));
      E4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (E)(acc[n][4 * k + i] * by);
      *reinterpret_cast<E4*>(to + 64 * n + 16 * k) = v;
    }
}

// Joins the parts of a tile's rows: workgroup (tile and head, y) every
// gridDim.y-th 256 / (D / 4) of them, D / 4 threads a row.
template <int D, bool kHalf>
__global__ __launch_bounds__(kPromptThreads) void prompt_join_kernel(PromptArgs a) {
  using E = typename Type16<kHalf>::E;
  constexpr int kAcross = D / 4, kRows = kPromptThreads / kAcross;
  PromptRows rows;
  Share share;
  if (!find_share<PromptTile<D>::kTokens, true>(a, blockIdx.x, rows, share) || share.chunks == 1)
    return;
  // (starts or lengths that change under the call)
  if ((uint32_t)share.first + (int64_t)(share.chunks - 1) * share.apart >= a.shares) return;
  const int head = share.head;
  const int c = (int)threadIdx.x % kAcross, in = (int)threadIdx.x / kAcross;
  const int pairs = min(rows.count * a.group - rows.tile * kTileRows, kTileRows);
  int key_first;
  bool bad;  // (never: such a row has no shares)
  const int pos0 = keys_of(a, rows, key_first, bad) - rows.count;
  for (int i = (int)blockIdx.y * kRows + in; in < kRows && i < pairs;
       i += kRows * (int)gridDim.y) {
    const int pair = rows.tile * kTileRows + i;
    const int64_t row = (int64_t)(rows.first + pair / a.group) * (a.heads * a.group) +
                        head * a.group + pair % a.group;
    float m = kNegInf, l = 0.0f;
    F32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto part_at = [&](uint32_t j) {
      return ((int64_t)share.first + (int64_t)j * share.apart) * kTileRows + i;
    };
    fold_parts<true>(
        0u, 1u, (uint32_t)share.chunks, m, l, o,
        [&](uint32_t j) { return a.part_ml[part_at(j)]; },
        [&](uint32_t j) {
          return *reinterpret_cast<const float4*>(a.part_acc + part_at(j) * D + 4 * c);
        });
    const float by = weight_of(pos0 + pair / a.group >= 0, l);
    typedef E E4 __attribute__((ext_vector_type(4)));
    E4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (E)(o[k] * by);
    *reinterpret_cast<E4*>(a.out + (row * D + 4 * c) * 2) = v;
  }
}

// Keys of a sequence: their numbers, and those of two tiles behind them, are ints.
constexpr int64_t kMostKeys = (int64_t(1) << 31) - 512;

struct PromptPlan {
  int tiles = 0, shares = 0, unit = 0;
  size_t acc_off = 0, total = 0;
};

// Tiles: at most those of all rows together and one more a sequence.  Where
// they leave half of the workgroups that the device holds at a time (two a CU)
// idle, that many share the tiles' keys.
PromptPlan prompt_plan(int64_t tokens, int64_t sequences, int64_t heads, int64_t group, int64_t dim,
                       int64_t most_keys) {
  PromptPlan P;
  const int64_t some = tokens < sequences ? tokens : sequences;
  P.tiles = (int)(tokens * group / kTileRows + some);
  const int64_t want = 2 * compute_units();
  if (P.tiles > 0 && P.tiles * heads * 2 <= want && most_keys > 256) {
    P.shares = (int)want;
    // (tiles times units are summed in 32 bits)
    while ((most_keys / 32 >> P.unit) + 2 > ((int64_t(1) << 32) - 1) / want) ++P.unit;
    const size_t rows = (size_t)want * kTileRows;
    P.acc_off = rows * sizeof(float2);
    P.total = P.acc_off + rows * dim * sizeof(float);
  }
  return P;
}

int check_prompt(const char* who, int dtype, int64_t tokens, int64_t sequences, int64_t heads,
                 int64_t group, int64_t dim) {
  if (dtype != RKV_BF16 && dtype != RKV_F16)
    return set_error(kUnsupported, "%s: rows must be bfloat16 or float16", who);
  if (!supported_dim(dim))
    return set_error(kUnsupported, "%s: head_dim %lld not in 32..256 step 32", who,
                     (long long)dim);
  const int64_t lim = (int64_t(1) << 31) - 1;
  if (tokens < 0 || sequences <= 0 || heads <= 0 || group <= 0 || sequences > lim ||
      heads > 65535 || group > 65535)
    return set_error(kInvalidArgument, "%s: empty or oversized shape", who);
  // (pairs of a sequence are counted in 32 bits, and so are a launch's threads)
  const int64_t most = (int64_t(1) << 32) / kPromptThreads - 1;
  if (tokens > lim / group - kTileRows || heads * group > lim ||
      (tokens * group / kTileRows + (tokens < sequences ? tokens : sequences) + 32) > most / heads)
    return set_error(kUnsupported, "%s: too many rows", who);
  return kOk;
}

int prompt(const char* who, PromptArgs& a, int dtype, int64_t tokens, int64_t sequences,
           int64_t heads, int64_t group, int64_t dim, int64_t most_keys, const void* query,
           int64_t q_ts, int64_t q_hs, float scale, const rkv_scores* scores, void* output,
           int zero_rest, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (tokens == 0) return kOk;
  if (!query || !output) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  q_ts = read_stride(q_ts, tokens);
  q_hs = read_stride(q_hs, heads * group);
  if (q_ts < 0 || q_hs < 0 || q_ts % 8 || q_hs % 8 || !aligned(query, 16) || !aligned(output, 16))
    return set_error(kInvalidArgument, "%s: query and output must be 16-byte aligned with strides "
                     "in multiples of 8", who);
  int rc = check_scores(who, scores);
  if (rc) return rc;
  const PromptPlan P = prompt_plan(tokens, sequences, heads, group, dim, most_keys);
  if (P.total) {
    if (!workspace || workspace_bytes < P.total)
      return set_error(kWorkspaceTooSmall, "%s: workspace of %zu bytes, %zu needed", who,
                       workspace_bytes, P.total);
    if (!aligned(workspace, 16))
      return set_error(kInvalidArgument, "%s: workspace must be 16-byte aligned", who);
    a.part_ml = static_cast<float2*>(workspace);
    a.part_acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + P.acc_off);
  }
  a.query = static_cast<const char*>(query);
  a.q_ts = q_ts;
  a.q_hs = q_hs;
  a.sequences = (int)sequences;
  a.heads = (int)heads;
  a.group = (int)group;
  a.tokens = (int)tokens;
  const float size = scale < 0.0f ? -scale : scale;
  a.scale = size * kLog2e;
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  a.window = scores_window(scores);
  if (scores) {
    a.slopes = scores->slopes;
    if (scores->softcap > 0.0f) {
      a.cap = scores->softcap * kLog2e;
      a.per_cap = size / scores->softcap;
    }
  }
  a.out = static_cast<char*>(output);
  // (rows behind the last sequence may be most of a padded batch: a workgroup for
  // every 256 of them, up to 32 a head)
  a.zero_rest = zero_rest ? (int)std::min<int64_t>(1 + tokens / 256, 32) : 0;
  a.tiles = P.tiles;
  a.shares = P.shares;
  a.unit = P.unit;
  // (a window alone changes no score; a scale of 0 times a hidden score would)
  const bool plain = !(a.cap > 0.0f) && !a.slopes && a.scale > 0.0f && a.scale < kPosInf;
  const int64_t blocks = P.shares ? P.shares : P.tiles * heads;
  // (the last workgroups: rows of no sequence)
  const dim3 grid((unsigned)(blocks + a.zero_rest * heads));
  const dim3 join((unsigned)(P.tiles * heads), 16), threads(kPromptThreads);
  RKV_DISPATCH_DIM(dim, D, {
    if (dtype == RKV_F16) {
      if (plain) prompt_kernel<D, true, false><<<grid, threads, 0, stream>>>(a);
      else prompt_kernel<D, true, true><<<grid, threads, 0, stream>>>(a);
      if (P.shares) prompt_join_kernel<D, true><<<join, threads, 0, stream>>>(a);
    } else {
      if (plain) prompt_kernel<D, false, false><<<grid, threads, 0, stream>>>(a);
      else prompt_kernel<D, false, true><<<grid, threads, 0, stream>>>(a);
      if (P.shares) prompt_join_kernel<D, false><<<join, threads, 0, stream>>>(a);
    }
  });
  return check_launch("prompt_kernel");
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_prompt_plan(int64_t tokens, int64_t sequences, int64_t heads, int64_t group,
                               int64_t dim, int64_t most_keys, size_t* workspace_bytes) {
  const char* who = "rkv_prompt_plan";
  clear_error();
  if (!workspace_bytes) return set_error(kInvalidArgument, "%s: null pointer", who);
  const int rc = check_prompt(who, RKV_BF16, tokens, sequences, heads, group, dim);
  if (rc) return rc;
  *workspace_bytes = prompt_plan(tokens, sequences, heads, group, dim, most_keys).total;
  return kOk;
}

extern "C" int rkv_prompt_attention(const void* query, int64_t q_token_stride,
                                    int64_t q_head_stride, const void* key, int64_t k_token_stride,
                                    int64_t k_head_stride, const void* value,
                                    int64_t v_token_stride, int64_t v_head_stride, int dtype,
                                    int64_t tokens, int64_t key_tokens, int64_t heads,
                                    int64_t group, int64_t dim, int64_t sequences,
                                    const int32_t* token_starts, const int32_t* key_starts,
                                    const int32_t* prefix, float scale, const rkv_scores* scores,
                                    void* output, int zero_rest, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
  const char* who = "rkv_prompt_attention";
  clear_error();
  int rc = check_prompt(who, dtype, tokens, sequences, heads, group, dim);
  if (rc) return rc;
  if (key_tokens < 0 || key_tokens > kMostKeys)
    return set_error(kInvalidArgument, "%s: bad key count", who);
  if (!token_starts && (sequences != 1 || key_starts))
    return set_error(kInvalidArgument, "%s: several sequences need token_starts", who);
  if (!key_starts && key_tokens != tokens)
    return set_error(kInvalidArgument, "%s: without key_starts as many keys as rows", who);
  if (tokens == 0) return kOk;
  if (key_tokens && (!key || !value))
    return set_error(kInvalidArgument, "%s: null pointer argument", who);
  PromptArgs a{};
  const int64_t strides[4] = {read_stride(k_token_stride, key_tokens),
                              read_stride(k_head_stride, heads),
                              read_stride(v_token_stride, key_tokens),
                              read_stride(v_head_stride, heads)};
  for (int64_t s : strides)
    if (s < 0 || s % 8)
      return set_error(kInvalidArgument, "%s: strides must be multiples of 8, not negative", who);
  if (!aligned(key, 16) || !aligned(value, 16))
    return set_error(kInvalidArgument, "%s: rows must be 16-byte aligned", who);
  // 16 rows are addressed with 32-bit byte offsets
  if (strides[0] > (1 << 25) || strides[2] > (1 << 25))
    return set_error(kUnsupported, "%s: rows more than 64 MiB apart", who);
  a.keys = static_cast<const char*>(key);
  a.values = static_cast<const char*>(value);
  a.k_ts = (uint32_t)(strides[0] * 2);
  a.k_hs = strides[1];
  a.v_ts = (uint32_t)(strides[2] * 2);
  a.v_hs = strides[3];
  a.key_tokens = (int)key_tokens;
  a.starts = token_starts;
  a.key_starts = key_starts;
  a.prefix = prefix;
  return prompt(who, a, dtype, tokens, sequences, heads, group, dim, key_tokens, query,
                q_token_stride, q_head_stride, scale, scores, output, zero_rest, workspace,
                workspace_bytes, stream);
}

extern "C" int rkv_paged_prompt(const rkv_paged_cache* cache, const void* query,
                                int64_t q_token_stride, int64_t q_head_stride, int64_t group,
                                int64_t tokens, const int32_t* token_starts,
                                const int32_t* prefix, float scale, const rkv_scores* scores,
                                void* output, int zero_rest, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  const char* who = "rkv_paged_prompt";
  clear_error();
  int rc = check_cache(who, cache);
  if (!rc)
    rc = check_prompt(who, cache->dtype, tokens, cache->sequences, cache->heads, group, cache->dim);
  if (rc) return rc;
  if (!token_starts && tokens != cache->sequences)
    return set_error(kInvalidArgument, "%s: without token_starts one token per sequence", who);
  if (cache->max_blocks * cache->page_size > kMostKeys)
    return set_error(kUnsupported, "%s: the block table covers too many tokens", who);
  PromptArgs a{};
  a.k_ps = read_stride(cache->key_page_stride, cache->pages);
  a.k_hs = read_stride(cache->key_head_stride, cache->heads);
  a.v_ps = read_stride(cache->value_page_stride, cache->pages);
  a.v_hs = read_stride(cache->value_head_stride, cache->heads);
  if (a.k_ps % 8 || a.k_hs % 8 || a.v_ps % 8 || a.v_hs % 8 || cache->key_token_stride % 8 ||
      cache->value_token_stride % 8 || !aligned(cache->keys, 16) || !aligned(cache->values, 16))
    return set_error(kInvalidArgument, "%s: the cache must be 16-byte aligned with strides in "
                     "multiples of 8", who);
  if (cache->key_token_stride > (1 << 25) || cache->value_token_stride > (1 << 25))
    return set_error(kUnsupported, "%s: rows more than 64 MiB apart", who);
  if (rows_meet_pages(cache, output, cache->heads * group * cache->dim, cache->dim, tokens,
                      cache->heads * group))
    return set_error(kInvalidArgument, "%s: output overlaps the cache", who);
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.k_ts = (uint32_t)(cache->key_token_stride * 2);
  a.v_ts = (uint32_t)(cache->value_token_stride * 2);
  a.starts = token_starts;
  a.step = !token_starts;
  a.lengths = cache->lengths;
  a.table = cache->block_table;
  a.table_stride = cache->table_stride;
  a.prefix = prefix;
  a.max_blocks = (int)cache->max_blocks;
  a.pages = (int)cache->pages;
  a.shift = page_shift(cache->page_size);
  return prompt(who, a, cache->dtype, tokens, cache->sequences, cache->heads, group, cache->dim,
                cache->max_blocks * cache->page_size, query, q_token_stride, q_head_stride, scale,
                scores, output, zero_rest, workspace, workspace_bytes, stream);
}
