// Attention of one new token per sequence over a paged KV cache:
//   out[b, h, g] = softmax_t(f(scale q[b, h, g] . K[t])) V,  t < lengths[b],
// token t of KV head h at row t % P of page table[b][t / P]; f is nothing, or
// caps the scores, biases them by distance and hides those before a window.
//
// Two launches: paged_kernel attends, paged_join_kernel joins the rows that
// several workgroups hold parts of.  (One launch whose last workgroup of a row
// joined it, through counters and stores past the caches, was as fast at best:
// one sequence of 2003 tokens 13.0 us against 12.5, of 131072 91.4 against
// 91.8, 128 short ones at head_dim 64 75 against 72.)  Sums, maxima and
// accumulators are fp32; the partition into shares depends on the batch's
// lengths and the device alone, so a call repeats bit for bit.
#include "rkv_paged_walk.h"

namespace rkv {
namespace {

// Workgroups per CU that share the tiles.  One keeps the CU's loads full (each
// of its waves has two tiles on their way) and leaves the fewest parts to
// join; at head_dim 32 a tile is 4 KB and two are needed.  From one to two: 32,
// 64 sequences of up to 20000 tokens 157 -> 129.5 us; 64, 128 of up to 2000
// 72.5 -> 72.2; 96, 32 of up to 8000 85.9 -> 87.9; 128, 131072 tokens 92.4 ->
// 94.0; 160, 24 of up to 4000 61.3 -> 67.7.
template <int D>
constexpr int kPerCu = D < 64 ? 2 : 1;

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

struct PagedArgs : WalkArgs {
  const char* keys;
  const char* values;
  int64_t k_ps, k_hs, v_ps, v_hs;  // page and head strides, elements
  uint32_t k_ts, v_ts;             // row strides, bytes
};

// The walk's operands from 16-bit pages: keys as they are stored, values
// transposed by byte permutes.
template <int D, bool kHalf_, bool kScores>
struct Pages16 {
  static constexpr int kDim = D;
  static constexpr bool kHalf = kHalf_, kScaleLate = false, kRareEnds = false;
  using Args = PagedArgs;
  using T = Type16<kHalf>;
  using V8 = typename T::V8;
  using E = typename T::E;
  using P = Pieces<D>;
  static constexpr int kAccs = P::kBlocks;

  // One tile's operands as they come from memory.
  struct Tile {
    U32x4 k[2][D / 32];
    U32x4 v8[P::k8 ? P::k8 : 1][8];
    U32x2 v4[8];
    uint32_t v2[8];
  };
  struct Query {
    V8 q[D / 32];
  };

  const Args& a;
  const int li, lg;
  const uint32_t ko;
  __device__ __forceinline__ Pages16(const Args& args, int li_, int lg_)
      : a(args), li(li_), lg(lg_), ko((uint32_t)li_ * args.k_ts + (uint32_t)lg_ * 16u) {}

  static __device__ __forceinline__ void take(Query& q, const U32x4 (&rows)[D / 32]) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) q.q[j] = __builtin_bit_cast(V8, rows[j]);
  }
  static __device__ __forceinline__ float unit(const Query&) { return 1.0f; }
  static __device__ __forceinline__ void finish(F32x4 (&)[kAccs]) {}

  // The loads of a tile, always as many (a tile or half that is not there
  // reads through an empty view): a later wait for one tile then never
  // waits for the next one's.
  __device__ __forceinline__ bool load(const Cursor& c, Tile& t, bool there) const {
    bool bad = c.bad;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = c.tile * kTileTokens + 16 * s;
      // rows of the half, those past the sequence's end left out
      const int rows = there ? min(c.length - at, 16) : 0;
      int page = s ? c.page1 : c.page0;
      const bool out = (uint32_t)page >= (uint32_t)a.pages;
      // (the pages of tokens that no query sees any more may be gone)
      bad |= out && rows > 0 && (!kScores || at + 15 >= c.length - a.window);
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
  }

  static __device__ __forceinline__ void scores(const Query& q, const Tile& t, float (&x)[8]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      F32x4 s4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < D / 32; ++j) s4 = T::mma(__builtin_bit_cast(V8, t.k[s][j]), q.q[j], s4);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[4 * s + r] = s4[r];
    }
  }

  // Whether any of the tile's values is infinite or NaN: its product with
  // zeros shows it as NaN.  (8 products more a tile at head_dim 128, on matrix
  // cores that wait for memory: 131072 tokens 91.6 -> 92.1 us, 2003 tokens
  // 11.85 -> 11.94, 128 short sequences at head_dim 64 71.6 -> 72.2.)
  static __device__ __forceinline__ bool has_infinite(const Tile& t) {
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
  }

  // Ones over the halves of a word that are infinite or NaN (the sum's top
  // bits: exponents of all ones).
  static __device__ __forceinline__ uint32_t infinite_of(uint32_t w) {
    const uint32_t top = (w & 0x7fff7fffu) + (kHalf ? 0x04000400u : 0x00800080u);
    return (top >> 15 & 0x00010001u) * 0xffffu;
  }

  // (tokens before `from` of the tile are hidden)
  __device__ __forceinline__ void products(F32x4 (&acc)[kAccs], Tile& t, const float (&p)[8],
                                           int from, int) const {
    if (kScores && from > 0) {
      // hidden tokens' values may be infinite or NaN: zeros here
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t seen = 16 * (e / 4) + 4 * lg + e % 4 >= from ? 0xffffffffu : 0u;
#pragma unroll
        for (int c8 = 0; c8 < P::k8; ++c8)
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v8[c8][e][i] &= seen;
        if constexpr (P::k4 > 0)
#pragma unroll
          for (int i = 0; i < 2; ++i) t.v4[e][i] &= seen;
        if constexpr (P::k2 > 0) t.v2[e] &= seen;
      }
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
};

// HBM bounds it: 8.6 GB of 16 x 131072 tokens (8 KV heads, group 4, d 128) in
// 1250-1325 us, 6.5-6.9 TB/s, by the card; the matrix cores are at 10 % and the
// vector ALUs at 15 %.  Small calls are a chain of latencies: 504 tiles of
// 2003 tokens take 7.2 us, of which 1.4 to know the share and its pages, 2.6
// until the first tile is done, 1.4 to join the waves; then 4.6 for the join
// kernel.
template <int D, bool kHalf, bool kScores>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void paged_kernel(PagedArgs a) {
  walk<Pages16<D, kHalf, kScores>, kScores>(a);
}

PagedPlan paged_plan(const rkv_paged_cache* c, int64_t group) {
  int grid = 0;
  RKV_DISPATCH_DIM(c->dim, D, grid = compute_units() * kPerCu<D>);
  return plan_of(grid, group, c->dim);
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

namespace {

int paged_decode(const char* who, const rkv_paged_cache* cache, const void* query,
                 int64_t q_sequence_stride, int64_t q_head_stride, int64_t group, float scale,
                 const rkv_scores* scores, void* output, void* workspace, size_t workspace_bytes,
                 hipStream_t stream) {
  clear_error();
  int rc = check_paged(who, cache, group);
  if (rc) return rc;
  PagedArgs a{};
  rc = walk_args(who, a, *cache, query, q_sequence_stride, q_head_stride, group, scale, scores,
                 output);
  if (rc) return rc;
  if (rows_meet_pages(cache, output, cache->heads * group * cache->dim, cache->dim,
                      cache->sequences, cache->heads * group))
    return set_error(kInvalidArgument, "%s: output overlaps the cache", who);
  const PagedPlan P = paged_plan(cache, group);
  rc = use_workspace(who, a, P, workspace, workspace_bytes);
  if (rc) return rc;
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.k_ps = read_stride(cache->key_page_stride, cache->pages);
  a.k_hs = read_stride(cache->key_head_stride, cache->heads);
  a.v_ps = read_stride(cache->value_page_stride, cache->pages);
  a.v_hs = read_stride(cache->value_head_stride, cache->heads);
  a.k_ts = (uint32_t)(cache->key_token_stride * 2);
  a.v_ts = (uint32_t)(cache->value_token_stride * 2);
  const dim3 grid((unsigned)P.grid), join((unsigned)P.grid, (unsigned)group);
  const bool plain = !scores_any(scores);
  const size_t parts = part_bytes(group, cache->dim);
  RKV_DISPATCH_DIM(cache->dim, D, {
    if (cache->dtype == RKV_F16) {
      if (plain) paged_kernel<D, true, false><<<grid, dim3(kThreads), parts, stream>>>(a);
      else paged_kernel<D, true, true><<<grid, dim3(kThreads), parts, stream>>>(a);
      paged_join_kernel<D, true><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    } else {
      if (plain) paged_kernel<D, false, false><<<grid, dim3(kThreads), parts, stream>>>(a);
      else paged_kernel<D, false, true><<<grid, dim3(kThreads), parts, stream>>>(a);
      paged_join_kernel<D, false><<<join, dim3(kJoinThreads), 0, stream>>>(a);
    }
  });
  return check_launch("paged_kernel");
}

}  // namespace

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
  return paged_decode("rkv_paged_decode", cache, query, q_sequence_stride, q_head_stride, group,
                      scale, nullptr, output, workspace, workspace_bytes, stream);
}

extern "C" int rkv_paged_decode_scores(const rkv_paged_cache* cache, const void* query,
                                       int64_t q_sequence_stride, int64_t q_head_stride,
                                       int64_t group, float scale, const rkv_scores* scores,
                                       void* output, void* workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
  return paged_decode("rkv_paged_decode_scores", cache, query, q_sequence_stride, q_head_stride,
                      group, scale, scores, output, workspace, workspace_bytes, stream);
}
