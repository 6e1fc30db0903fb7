// Attention of one new token per sequence over a paged KV cache:
//   out[b, h, g] = softmax_t(scale q[b, h, g] . K[t]) V,  t < lengths[b],
// token t of KV head h at row t % P of page table[b][t / P].
#include "rkv_common.h"
#include "rkv_internal.h"
#include "rkv_paged.h"

namespace rkv {
namespace {

constexpr int kThreads = 256;

struct PagedArgs {
  const char* query;             // (B, H G, D), strides in elements
  int64_t q_bs, q_hs;
  const char* keys;
  const char* values;
  int64_t k_ps, k_hs, k_ts;      // page, head and token strides, elements
  int64_t v_ps, v_hs, v_ts;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  int sequences, heads, group, max_blocks, pages, shift;
  float scale;
  char* out;                     // (B, H G, D) dense
};

template <bool kHalf>
__device__ __forceinline__ float load16(const char* p) {
  if constexpr (kHalf) return (float)*reinterpret_cast<const _Float16*>(p);
  return bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
}

// One workgroup per (query head, sequence): 16 lanes share a token's dims, 16
// such groups take every 16th token with a running maximum and sum, joined at
// the end in LDS.
template <int D, bool kHalf>
__global__ __launch_bounds__(kThreads) void paged_kernel(PagedArgs a) {
  constexpr int CH = D / 16;
  __shared__ float acc_s[16][D];
  __shared__ float m_s[16], l_s[16];
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / a.group;
  const int c = threadIdx.x % 16, grp = threadIdx.x / 16;
  const int length = a.lengths[b];
  const char* q = a.query + (b * a.q_bs + hq * a.q_hs + c * CH) * 2;
  float qf[CH], acc[CH];
  for (int i = 0; i < CH; ++i) {
    qf[i] = load16<kHalf>(q + 2 * i);
    acc[i] = 0.0f;
  }
  float m = kNegInf, l = 0.0f;
  bool bad = length > a.max_blocks << a.shift;
  for (int t = grp; t < length && !bad; t += 16) {
    const int page = a.table[b * a.table_stride + (t >> a.shift)];
    if (page < 0 || page >= a.pages) {
      bad = true;
      break;
    }
    const int64_t row = t & ((1 << a.shift) - 1);
    const char* k = a.keys + (page * a.k_ps + h * a.k_hs + row * a.k_ts + c * CH) * 2;
    const char* v = a.values + (page * a.v_ps + h * a.v_hs + row * a.v_ts + c * CH) * 2;
    float s = 0.0f;
    for (int i = 0; i < CH; ++i) s = __builtin_fmaf(qf[i], load16<kHalf>(k + 2 * i), s);
    s = row16_sum_all(s) * a.scale;
    const float mn = nanmax(m, s);
    const float w = m == mn ? 1.0f : exp_hw(m - mn);
    const float p = s == kNegInf ? 0.0f : exp_hw(s - mn);
    l = l * w + p;
    for (int i = 0; i < CH; ++i)
      acc[i] = __builtin_fmaf(p, load16<kHalf>(v + 2 * i), acc[i] * w);
    m = mn;
  }
  if (bad) l = __builtin_nanf("");
  for (int i = 0; i < CH; ++i) acc_s[grp][c * CH + i] = acc[i];
  if (c == 0) {
    m_s[grp] = m;
    l_s[grp] = l;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  float M = kNegInf;
  for (int j = 0; j < 16; ++j) M = nanmax(M, m_s[j]);
  float L = 0.0f, o = 0.0f;
  for (int j = 0; j < 16; ++j) {
    if (l_s[j] == 0.0f) continue;
    const float w = m_s[j] == M ? 1.0f : exp_hw(m_s[j] - M);
    L += l_s[j] * w;
    o += acc_s[j][d] * w;
  }
  const float y = length <= 0 ? 0.0f : o / L;
  char* out = a.out + (((int64_t)b * a.heads * a.group + hq) * D + d) * 2;
  if constexpr (kHalf) *reinterpret_cast<_Float16*>(out) = (_Float16)y;
  else *reinterpret_cast<uint16_t*>(out) = bf16_rne(y);
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
  const int64_t strides[] = {c->key_page_stride, c->key_head_stride, c->key_token_stride,
                             c->value_page_stride, c->value_head_stride, c->value_token_stride};
  for (int64_t s : strides)
    if (s % 8) return set_error(kInvalidArgument, "%s: cache strides must be multiples of 8", who);
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
  *workspace_bytes = 0;
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
  if (!aligned(query, 16) || !aligned(output, 16) || q_sequence_stride % 8 || q_head_stride % 8)
    return set_error(kInvalidArgument,
                     "%s: query and output must be 16-byte aligned with strides in multiples of 8",
                     who);
  PagedArgs a{};
  a.query = static_cast<const char*>(query);
  a.q_bs = q_sequence_stride;
  a.q_hs = q_head_stride;
  a.keys = static_cast<const char*>(cache->keys);
  a.values = static_cast<const char*>(cache->values);
  a.k_ps = cache->key_page_stride;
  a.k_hs = cache->key_head_stride;
  a.k_ts = cache->key_token_stride;
  a.v_ps = cache->value_page_stride;
  a.v_hs = cache->value_head_stride;
  a.v_ts = cache->value_token_stride;
  a.table = cache->block_table;
  a.table_stride = cache->table_stride;
  a.lengths = cache->lengths;
  a.sequences = (int)cache->sequences;
  a.heads = (int)cache->heads;
  a.group = (int)group;
  a.max_blocks = (int)cache->max_blocks;
  a.pages = (int)cache->pages;
  a.shift = page_shift(cache->page_size);
  a.scale = scale;
  a.out = static_cast<char*>(output);
  const dim3 grid((unsigned)(cache->heads * group), (unsigned)cache->sequences);
  const bool half = cache->dtype == RKV_F16;
  RKV_DISPATCH_DIM(cache->dim, D, {
    if (half) paged_kernel<D, true><<<grid, dim3(kThreads), 0, stream>>>(a);
    else paged_kernel<D, false><<<grid, dim3(kThreads), 0, stream>>>(a);
  });
  return check_launch("paged_kernel");
}
