// Rotary positions, alone (rkv_rotary) and on the way into a paged KV cache
// (rkv_paged_append).
//
// A pair (x0, x1) of a head's rotated part turns by t = position * rate_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,  c = a cos t, s = a sin t,
// with a the table's attention factor.  The half layout pairs dims i and
// i + r/2, the interleaved one 2i and 2i + 1; dims from r on pass.  Memory
// bound: every value is read and written once, at 5.9 TB/s for long prompts
// (131001 tokens of 32 + 8 + 8 heads, d 128, 3.2 GB: 542 us; torch's copy of
// 2 GiB reaches 5.0 TB/s).  A cos and sin costs some 30 instructions a pair
// (45 before the quarters were taken off by one addition), so a thread that
// turned one head alone was bound by them (862 us).
#include "rkv_common.h"
#include "rkv_internal.h"
#include "rkv_paged.h"
#include "rkv_places.h"

namespace rkv {
namespace {

constexpr int kThreads = 256;
// Heads of a thread's loads in flight together (1, 3 and 4 instead of 2: 64 K
// tokens of 28 + 4 heads 187, 185 and 181 us against 183, 131001 tokens of 48
// heads 553, 561 and 546 against 541, 24 K ragged ones of 36 heads 37, 38 and
// 41 against 36, eight tokens of 40 heads 4.1, 4.5 and 4.8 against 4.0).
constexpr int kBatch = 2;
// A call that writes more than the last-level cache holds (256 MB) stores past
// it; what a smaller one writes is left there for whoever reads it next.
// Rotation of 28 + 4 heads, in parentheses with an elementwise kernel that then
// reads the queries, us by bytes written: stored past the cache and not, 64 MB
// 27.1 (46.9) and 26.8 (44.2), 128 MB 49.1 (85.2) and 47.5 (80.4), 192 MB 70.6
// (123) and 66.5 (119), 256 MB 92.9 (176) and 86.5 (180), 384 MB 137 (258) and
// 150 (268), 512 MB 182 (340) and 199 (357).
constexpr int64_t kStreamBytes = int64_t(256) << 20;
// From so many threads on the device is full (4 waves per SIMD), and fewer
// threads turn more heads each with the same cos and sin.
constexpr int64_t kManyThreads = 4 * 1024 * 64;

// A set of rows (token, head, dim): strides in elements, dim dense.
struct Rows {
  const char* src;
  char* dst;                 // rows, or the cache's pages for keys and values
  int64_t src_ts, src_hs;    // token and head strides of src, elements
  int64_t dst_ts, dst_hs;    // of dst (a page's row and head strides in a cache)
  int64_t dst_ps;            // page stride of dst, elements (cache only)
  int heads;
  int paged;                 // dst is the cache's pages (keys and values alike)
};

struct RotaryArgs : Places {
  Rows rows[3];              // queries, keys, values (heads 0: absent)
  int heads;                 // all of them
  int64_t tokens;
  int dim, rotary_dim;
  const double* rates;       // turns per position of each pair, rotary_dim / 2
  float scale, sign;         // attention factor; -1 turns back
  int items, turning;        // items of a head's row; those that turn come first
  int step, gap;             // dims from one turning item to the next, of an item's two vectors
  int slots, per_block;      // heads that a token's threads hold at a time, a workgroup's tokens
};

// One of three values, chosen as values: a choice between variables would be
// one of addresses, and put them in scratch.
template <typename T>
__device__ __forceinline__ T pick(bool q, bool v, T of_query, T of_key, T of_value) {
  return q ? of_query : v ? of_value : of_key;
}

// A thread holds one item of a row, two vectors of W dims: in the half layout
// r/2 apart (W pairs), in the interleaved one side by side (kAdjacent: W / 2
// pairs each; W 1: one pair), and side by side too where dims pass.  A part
// that is an odd number of vectors has one in its last item.  (One vector an
// item where dims pass: 50266 tokens of 28 + 4 heads, 64 of 128 dims turning,
// 207 us against 182.)  The thread works out the item's cos and sin once and
// applies them to every slots-th head of its token, kBatch heads at a time
// whose loads are all in flight before the first use; those of the first
// batch are on their way before the position is known.
template <typename T, int W, bool kAdjacent, bool kStream>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int kPairs = W;
  constexpr int kSize = sizeof(T);
  typedef T V __attribute__((ext_vector_type(W)));
  const int wide = a.items < kThreads ? a.items : kThreads;
  const int in_block = (int)(threadIdx.x / (uint32_t)(wide * a.slots));
  const uint32_t rest = threadIdx.x % (uint32_t)(wide * a.slots);
  const int slot = (int)(rest / (uint32_t)wide);
  const int64_t t = (int64_t)blockIdx.x * a.per_block + in_block;
  if (in_block >= a.per_block || t >= a.tokens) return;
  Place place;
  bool placed = false;
  for (int item = (int)(rest % (uint32_t)wide); item < a.items; item += kThreads) {
    const bool turns = item < a.turning;
    const int d0 = turns ? item * a.step : a.rotary_dim + (item - a.turning) * (2 * W);
    const int gap = turns ? a.gap : W;
    const bool two = turns ? !kAdjacent || d0 + W < a.rotary_dim : d0 + W < a.dim;
    V x[kBatch], z[kBatch];
    // queries, then keys, then values: each kind's first head, and the others
    // by its head stride
    const int q_end = a.rows[0].heads, k_end = q_end + a.rows[1].heads;
    const char* const from_q = a.rows[0].src + (t * a.rows[0].src_ts + d0) * kSize;
    const char* const from_k = a.rows[1].src + (t * a.rows[1].src_ts + d0) * kSize;
    const char* const from_v = a.rows[2].src + (t * a.rows[2].src_ts + d0) * kSize;
    const int64_t q_hs = a.rows[0].src_hs * kSize, k_hs = a.rows[1].src_hs * kSize,
                  v_hs = a.rows[2].src_hs * kSize;
    auto load = [&](int n0) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int n = min(n0 + i * a.slots, a.heads - 1);
        const bool q = n < q_end, v = n >= k_end;
        const int h = n - (q ? 0 : v ? k_end : q_end);
        const char* src = pick(q, v, from_q, from_k, from_v) + h * pick(q, v, q_hs, k_hs, v_hs);
        x[i] = __builtin_nontemporal_load(reinterpret_cast<const V*>(src));
        if (two)
          z[i] = __builtin_nontemporal_load(reinterpret_cast<const V*>(src + gap * kSize));
      }
    };
    load(slot);
    if (!placed) place = place_of(a, t);
    placed = true;
    const bool live = turns && place.live;
    const double position4 = 4.0 * (double)place.position;  // rates are whole turns
    float c[kPairs], s[kPairs];
    if (live) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        // (the pairs of a second vector that is not there are not read)
        const int pair = item * kPairs + (kAdjacent && i >= W / 2 && !two ? 0 : i);
        cos_sin(position4 * a.rates[pair], c[i], s[i]);
        c[i] *= a.scale;
        s[i] *= a.scale * a.sign;
      }
    }
    // (a cache's keys and values, or rows of this token)
    const int64_t k_row = a.rows[1].paged ? place.page * a.rows[1].dst_ps +
                                                place.row * a.rows[1].dst_ts
                                          : t * a.rows[1].dst_ts;
    const int64_t v_row = place.page * a.rows[2].dst_ps + place.row * a.rows[2].dst_ts;
    char* const to_q = a.rows[0].dst + (t * a.rows[0].dst_ts + d0) * kSize;
    char* const to_k = a.rows[1].dst + (k_row + d0) * kSize;
    char* const to_v = a.rows[2].dst + (v_row + d0) * kSize;
    const int64_t qo_hs = a.rows[0].dst_hs * kSize, ko_hs = a.rows[1].dst_hs * kSize,
                  vo_hs = a.rows[2].dst_hs * kSize;
    const bool stored = place.page >= 0;  // keys and values of a cache
    for (int n0 = slot;;) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int n = n0 + i * a.slots;
        const bool q = n < q_end, v = n >= k_end;
        const int h = n - (q ? 0 : v ? k_end : q_end);
        if (n >= a.heads || (!q && a.rows[1].paged && !stored)) continue;
        if (live && !v) {
#pragma unroll
          for (int p = 0; p < kPairs; ++p) {
            float x0, x1;
            V& pairs = p < W / 2 ? x[i] : z[i];
            const int at = p % (W / 2 > 0 ? W / 2 : 1) * 2;
            if constexpr (kAdjacent) x0 = (float)pairs[at], x1 = (float)pairs[at + 1];
            else x0 = (float)x[i][p], x1 = (float)z[i][p];
            const float y0 = __builtin_fmaf(x0, c[p], -(x1 * s[p]));
            const float y1 = __builtin_fmaf(x1, c[p], x0 * s[p]);
            if constexpr (kAdjacent) {
              pairs[at] = (T)y0;
              pairs[at + 1] = (T)y1;
            } else {
              x[i][p] = (T)y0;
              z[i][p] = (T)y1;
            }
          }
        }
        char* dst = pick(q, v, to_q, to_k, to_v) + h * pick(q, v, qo_hs, ko_hs, vo_hs);
        V* const to_x = reinterpret_cast<V*>(dst);
        V* const to_z = reinterpret_cast<V*>(dst + gap * kSize);
        if constexpr (kStream) {
          __builtin_nontemporal_store(x[i], to_x);
          if (two) __builtin_nontemporal_store(z[i], to_z);
        } else {
          *to_x = x[i];
          if (two) *to_z = z[i];
        }
      }
      n0 += kBatch * a.slots;
      if (n0 >= a.heads) break;
      load(n0);
    }
  }
}

// Bytes of the widest vector (16, 8 or one element) that every row's address
// and the rotated and passing parts allow.
int vector_bytes(const RotaryArgs& a, int size, bool interleaved) {
  const int64_t half = (int64_t)a.rotary_dim / 2;
  for (int bytes = 16; bytes > size; bytes >>= 1) {
    const int64_t n = bytes / size;
    if (bytes < 8 || (interleaved ? a.rotary_dim : half) % n || (a.dim - a.rotary_dim) % n)
      continue;
    bool ok = true;
    for (const Rows& r : a.rows) {
      if (!r.heads) continue;
      ok = ok && aligned(r.src, bytes) && aligned(r.dst, bytes) && r.src_ts % n == 0 &&
           r.src_hs % n == 0 && r.dst_ts % n == 0 && r.dst_hs % n == 0 && r.dst_ps % n == 0;
    }
    if (ok) return bytes;
  }
  return size;
}

template <typename T, int W, bool kAdjacent>
int launch_w(RotaryArgs& a, hipStream_t stream) {
  const int half = a.rotary_dim / 2;
  a.turning = kAdjacent ? (half + W - 1) / W : half / W;
  a.items = a.turning + (a.dim - a.rotary_dim + 2 * W - 1) / (2 * W);
  const int wide = a.items < kThreads ? a.items : kThreads;
  // Few tokens: every thread kBatch heads, for latency.  Many: a wave holds
  // one token's consecutive heads (d 128: 8 heads, 2 KB), each thread every
  // 8th of them (against every 4th and 16th, 64 K tokens of 28 + 4 heads: 183
  // against 197 and 192 us, 131001 of 48 heads 541 against 584 and 553).
  a.slots = (a.heads + kBatch - 1) / kBatch;
  if (a.tokens * wide * a.slots >= kManyThreads) a.slots = wide < kWave ? kWave / wide : 1;
  a.slots = a.slots < a.heads ? a.slots : a.heads;
  a.slots = a.slots < kThreads / wide ? a.slots : kThreads / wide;
  a.per_block = kThreads / (wide * a.slots);
  const int64_t blocks = (a.tokens + a.per_block - 1) / a.per_block;
  if (!launch_fits(blocks, kThreads))
    return set_error(kInvalidArgument, "rotary: too many tokens");
  const int64_t bytes = a.tokens * a.heads * a.dim * (int64_t)sizeof(T);
  if (bytes >= kStreamBytes)
    rotary_kernel<T, W, kAdjacent, true><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a);
  else
    rotary_kernel<T, W, kAdjacent, false><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a);
  return check_launch("rotary_kernel");
}

template <typename T>
int launch_t(RotaryArgs& a, bool interleaved, hipStream_t stream) {
  constexpr int kSize = sizeof(T);
  const int bytes = vector_bytes(a, kSize, interleaved);
  if (interleaved && bytes > kSize) {
    a.gap = bytes / kSize;
    a.step = 2 * a.gap;
    return bytes == 16 ? launch_w<T, 16 / kSize, true>(a, stream)
                       : launch_w<T, 8 / kSize, true>(a, stream);
  }
  a.gap = interleaved ? 1 : a.rotary_dim / 2;
  a.step = interleaved ? 2 : bytes / kSize;
  if (bytes == 16) return launch_w<T, 16 / kSize, false>(a, stream);
  if (bytes == 8) return launch_w<T, 8 / kSize, false>(a, stream);
  return launch_w<T, 1, false>(a, stream);
}

int launch(RotaryArgs& a, int dtype, bool interleaved, hipStream_t stream) {
  a.heads = 0;
  for (const Rows& r : a.rows) a.heads += r.heads;
  if (a.tokens == 0 || a.heads == 0) return kOk;
  if (dtype == RKV_BF16) return launch_t<__bf16>(a, interleaved, stream);
  if (dtype == RKV_F16) return launch_t<_Float16>(a, interleaved, stream);
  return launch_t<float>(a, interleaved, stream);
}

// Rows of a cache's pages copied out, `bytes` of a vector at a time.
struct ReadArgs : Places {
  const char* src[2];           // keys, values
  char* dst[2];                 // (tokens, heads, dim) dense
  int64_t ps[2], hs[2], ts[2];  // page, head and row strides of src, bytes
  int64_t tokens;
  int heads, row_bytes, dtype;
};

template <typename V>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(ReadArgs a) {
  const int items = a.row_bytes / (int)sizeof(V), each = 2 * a.heads * items;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t t = id / each;
  if (t >= a.tokens) return;
  const int rest = (int)(id % each);
  const int item = rest % items, h = rest / items % a.heads, k = rest / items / a.heads;
  const Place p = place_of(a, t);
  V v{};
  if (p.page >= 0) {
    v = *reinterpret_cast<const V*>((k ? a.src[1] : a.src[0]) +
                                    p.page * (k ? a.ps[1] : a.ps[0]) +
                                    h * (k ? a.hs[1] : a.hs[0]) +
                                    p.row * (k ? a.ts[1] : a.ts[0]) + item * sizeof(V));
  } else if (p.live) {
    // NaN of the type, in every element of the vector
    const uint32_t nan = a.dtype == RKV_F32    ? 0x7fc00000u
                         : a.dtype == RKV_BF16 ? 0x7fc07fc0u
                                               : 0x7e007e00u;
    __builtin_memcpy(&v, &nan, sizeof(V) < 4 ? sizeof(V) : 4);
    if constexpr (sizeof(V) > 4)
      for (size_t i = 4; i < sizeof(V); i += 4)
        __builtin_memcpy(reinterpret_cast<char*>(&v) + i, &nan, 4);
  }
  *reinterpret_cast<V*>((k ? a.dst[1] : a.dst[0]) + (t * a.heads + h) * a.row_bytes +
                        item * (int64_t)sizeof(V)) = v;
}

template <typename V>
int launch_read(const ReadArgs& a, hipStream_t stream) {
  const int64_t each = 2 * (int64_t)a.heads * (a.row_bytes / (int)sizeof(V));
  const bool fits = launch_fits(a.tokens, each);
  const int64_t blocks = fits ? (a.tokens * each + kThreads - 1) / kThreads : 0;
  if (!fits || !launch_fits(blocks, kThreads))
    return set_error(kInvalidArgument, "rkv_paged_read: too many tokens");
  paged_read_kernel<V><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a);
  return check_launch("paged_read_kernel");
}

int check_table(const char* who, const double* rates, int64_t rotary_dim, int64_t dim) {
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > dim || (rotary_dim > 0 && !rates))
    return set_error(kInvalidArgument, "%s: rotary_dim %lld must be even, at most head_dim %lld, "
                     "with its rates", who, (long long)rotary_dim, (long long)dim);
  return kOk;
}

int check_rows(const char* who, const void* src, const void* dst, int64_t heads, int size) {
  if (heads < 0 || heads > 65535) return set_error(kInvalidArgument, "%s: bad head count", who);
  if (heads && (!src || !dst)) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  if (heads && (!aligned(src, size) || !aligned(dst, size)))
    return set_error(kInvalidArgument, "%s: rows not aligned to their type", who);
  return kOk;
}

Rows plain_rows(int64_t tokens, const void* src, int64_t ts, int64_t hs, int64_t heads, void* dst,
                int64_t dst_ts, int64_t dst_hs) {
  Rows r{};
  r.src = static_cast<const char*>(src);
  r.dst = static_cast<char*>(dst);
  r.src_ts = read_stride(ts, tokens);
  r.src_hs = read_stride(hs, heads);
  r.dst_ts = read_stride(dst_ts, tokens);
  r.dst_hs = read_stride(dst_hs, heads);
  r.heads = (int)heads;
  return r;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_rotary(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                          int64_t q_heads, const void* key, int64_t k_token_stride,
                          int64_t k_head_stride, int64_t k_heads, int dtype, int64_t tokens,
                          int64_t dim, const void* positions, int wide_positions,
                          const double* rates, int64_t rotary_dim, int interleaved, float scale,
                          int inverse, void* query_out, int64_t qo_token_stride,
                          int64_t qo_head_stride, void* key_out, int64_t ko_token_stride,
                          int64_t ko_head_stride, hipStream_t stream) {
  const char* who = "rkv_rotary";
  clear_error();
  if (!known_dtype(dtype)) return set_error(kUnsupported, "%s: dtype %d", who, dtype);
  if (tokens < 0 || dim <= 0 || dim > 65535)
    return set_error(kInvalidArgument, "%s: bad shape", who);
  if (tokens && !positions) return set_error(kInvalidArgument, "%s: null positions", who);
  const int size = (int)dtype_bytes(dtype);
  int rc = check_table(who, rates, rotary_dim, dim);
  if (!rc) rc = check_rows(who, query, query_out, tokens ? q_heads : 0, size);
  if (!rc) rc = check_rows(who, key, key_out, tokens ? k_heads : 0, size);
  if (rc) return rc;
  RotaryArgs a{};
  a.rows[0] = plain_rows(tokens, query, q_token_stride, q_head_stride, q_heads, query_out,
                         qo_token_stride, qo_head_stride);
  a.rows[1] = plain_rows(tokens, key, k_token_stride, k_head_stride, k_heads, key_out, ko_token_stride,
                         ko_head_stride);
  a.tokens = tokens;
  a.dim = (int)dim;
  a.rotary_dim = (int)rotary_dim;
  a.positions = positions;
  a.wide_positions = wide_positions;
  a.rates = rates;
  a.scale = scale;
  a.sign = inverse ? -1.0f : 1.0f;
  return launch(a, dtype, interleaved != 0, stream);
}

extern "C" int rkv_paged_append(const rkv_paged_cache* cache, const void* query,
                                int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                                void* query_out, int64_t qo_token_stride, int64_t qo_head_stride,
                                const void* key, int64_t k_token_stride, int64_t k_head_stride,
                                const void* value, int64_t v_token_stride, int64_t v_head_stride,
                                int64_t tokens, const int32_t* token_starts, const double* rates,
                                int64_t rotary_dim, int interleaved, float scale,
                                hipStream_t stream) {
  const char* who = "rkv_paged_append";
  clear_error();
  int rc = check_cache(who, cache);
  if (rc) return rc;
  if (tokens < 0 || (!token_starts && tokens != cache->sequences))
    return set_error(kInvalidArgument, "%s: without token_starts one token per sequence", who);
  const int size = (int)dtype_bytes(cache->dtype);
  rc = check_table(who, rates, rotary_dim, cache->dim);
  if (!rc) rc = check_rows(who, query, query_out, tokens ? q_heads : 0, size);
  if (!rc) rc = check_rows(who, key, cache->keys, tokens ? cache->heads : 0, size);
  if (!rc) rc = check_rows(who, value, cache->values, tokens ? cache->heads : 0, size);
  if (rc) return rc;
  if (keys_meet_values(cache))
    return set_error(kInvalidArgument, "%s: the cache's keys and values share memory", who);
  if (q_heads && rows_meet_pages(cache, query_out, qo_token_stride, qo_head_stride, tokens, q_heads))
    return set_error(kInvalidArgument, "%s: query_out overlaps the cache", who);
  if (rows_meet_pages(cache, key, k_token_stride, k_head_stride, tokens, cache->heads) ||
      rows_meet_pages(cache, value, v_token_stride, v_head_stride, tokens, cache->heads) ||
      (q_heads && rows_meet_pages(cache, query, q_token_stride, q_head_stride, tokens, q_heads)))
    return set_error(kRowsInCache, "%s: rows overlap the cache", who);
  RotaryArgs a{};
  a.rows[0] = plain_rows(tokens, query, q_token_stride, q_head_stride, q_heads, query_out,
                         qo_token_stride, qo_head_stride);
  a.rows[1] = plain_rows(tokens, key, k_token_stride, k_head_stride, cache->heads, cache->keys,
                         cache->key_token_stride, cache->key_head_stride);
  a.rows[2] = plain_rows(tokens, value, v_token_stride, v_head_stride, cache->heads, cache->values,
                         cache->value_token_stride, cache->value_head_stride);
  a.rows[1].dst_ts = cache->key_token_stride;  // of a page's rows, however few tokens come
  a.rows[2].dst_ts = cache->value_token_stride;
  a.rows[1].dst_ps = read_stride(cache->key_page_stride, cache->pages);
  a.rows[2].dst_ps = read_stride(cache->value_page_stride, cache->pages);
  a.rows[1].paged = a.rows[2].paged = 1;
  a.tokens = tokens;
  a.dim = (int)cache->dim;
  a.rotary_dim = (int)rotary_dim;
  a.rates = rates;
  a.scale = scale;
  a.sign = 1.0f;
  a.starts = token_starts;
  a.lengths = cache->lengths;
  a.table = cache->block_table;
  a.table_stride = cache->table_stride;
  a.sequences = (int)cache->sequences;
  a.max_blocks = (int)cache->max_blocks;
  a.pages = (int)cache->pages;
  a.shift = page_shift(cache->page_size);
  return launch(a, cache->dtype, interleaved != 0, stream);
}

extern "C" int rkv_paged_read(const rkv_paged_cache* cache, int64_t tokens,
                              const int32_t* token_starts, void* key_out, void* value_out,
                              hipStream_t stream) {
  const char* who = "rkv_paged_read";
  clear_error();
  const int rc = check_cache(who, cache);
  if (rc) return rc;
  if (tokens < 0 || (!token_starts && tokens != cache->sequences))
    return set_error(kInvalidArgument, "%s: without token_starts one token per sequence", who);
  if (tokens == 0) return kOk;
  if (!key_out || !value_out) return set_error(kInvalidArgument, "%s: null pointer argument", who);
  const int64_t size = dtype_bytes(cache->dtype), row = cache->heads * cache->dim;
  if (!aligned(key_out, size) || !aligned(value_out, size))
    return set_error(kInvalidArgument, "%s: rows not aligned to their type", who);
  const uint64_t k0 = reinterpret_cast<uint64_t>(key_out), v0 = reinterpret_cast<uint64_t>(value_out);
  const uint64_t bytes = (uint64_t)(tokens * row * size);
  if (rows_meet_pages(cache, key_out, row, cache->dim, tokens, cache->heads) ||
      rows_meet_pages(cache, value_out, row, cache->dim, tokens, cache->heads) ||
      (k0 < v0 + bytes && v0 < k0 + bytes))
    return set_error(kInvalidArgument, "%s: the rows overlap each other or the cache", who);
  ReadArgs a{};
  a.src[0] = static_cast<const char*>(cache->keys);
  a.src[1] = static_cast<const char*>(cache->values);
  a.dst[0] = static_cast<char*>(key_out);
  a.dst[1] = static_cast<char*>(value_out);
  a.ps[0] = read_stride(cache->key_page_stride, cache->pages) * size;
  a.ps[1] = read_stride(cache->value_page_stride, cache->pages) * size;
  a.hs[0] = read_stride(cache->key_head_stride, cache->heads) * size;
  a.hs[1] = read_stride(cache->value_head_stride, cache->heads) * size;
  a.ts[0] = cache->key_token_stride * size;
  a.ts[1] = cache->value_token_stride * size;
  a.tokens = tokens;
  a.heads = (int)cache->heads;
  a.row_bytes = (int)(cache->dim * size);
  a.dtype = cache->dtype;
  a.starts = token_starts;
  a.lengths = cache->lengths;
  a.table = cache->block_table;
  a.table_stride = cache->table_stride;
  a.sequences = (int)cache->sequences;
  a.max_blocks = (int)cache->max_blocks;
  a.pages = (int)cache->pages;
  a.shift = page_shift(cache->page_size);
  // the widest vector that every row's address allows
  int64_t all = a.row_bytes;
  for (int i = 0; i < 2; ++i)
    all |= (int64_t)reinterpret_cast<uint64_t>(a.src[i]) | (int64_t)reinterpret_cast<uint64_t>(a.dst[i]) |
           a.ps[i] | a.hs[i] | a.ts[i];
  if (all % 16 == 0) return launch_read<uint4>(a, stream);
  if (all % 4 == 0) return launch_read<uint32_t>(a, stream);
  return launch_read<uint16_t>(a, stream);
}
