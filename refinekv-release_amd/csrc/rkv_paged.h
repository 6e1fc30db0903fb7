// What the paged-cache entry points share: the checked view of a caller's
// rkv_paged_cache and the host-side checks of it.
#pragma once

#include "../../include/refinekv_hip.h"
#include "rkv_internal.h"

namespace rkv {

inline int64_t dtype_bytes(int dtype) { return dtype == RKV_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == RKV_BF16 || dtype == RKV_F16 || dtype == RKV_F32; }

// log2 of a supported page size (16, 32, 64, 128 or 256 tokens), else -1.
inline int page_shift(int64_t page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (int64_t(1) << s)) return s;
  return -1;
}

// The checks every entry makes of a cache.  Pages are numbered in int32 and
// positions are int32, so both counts are bounded by it; the addresses made
// of them are 64-bit.
inline int check_cache(const char* who, const rkv_paged_cache* c) {
  const int64_t lim = (int64_t(1) << 31) - 1;
  if (!c) return set_error(kInvalidArgument, "%s: null cache", who);
  if (!c->keys || !c->values || !c->block_table || !c->lengths)
    return set_error(kInvalidArgument, "%s: null pointer in the cache", who);
  if (!known_dtype(c->dtype)) return set_error(kUnsupported, "%s: dtype %d", who, c->dtype);
  if (c->pages <= 0 || c->heads <= 0 || c->dim <= 0 || c->sequences <= 0 || c->max_blocks <= 0 ||
      c->pages > lim || c->heads > 65535 || c->dim > 65535 || c->sequences > lim)
    return set_error(kInvalidArgument, "%s: empty or oversized cache", who);
  if (page_shift(c->page_size) < 0)
    return set_error(kUnsupported, "%s: page_size %lld not in {16, 32, 64, 128, 256}", who,
                     (long long)c->page_size);
  if (c->max_blocks > lim / c->page_size)
    return set_error(kInvalidArgument, "%s: the block table covers 2^31 tokens or more", who);
  if (c->table_stride < 0 || c->key_page_stride < 0 || c->key_head_stride < 0 ||
      c->key_token_stride < 0 || c->value_page_stride < 0 || c->value_head_stride < 0 ||
      c->value_token_stride < 0)
    return set_error(kInvalidArgument, "%s: negative stride", who);
  return kOk;
}

// An axis of a cache: strides in bytes, and its places.
struct CacheAxis {
  int64_t key, value, count;
};

// Whether keys and values from axis `level` on share a cell, the values' first
// one `apart` behind the keys'.  Axes go from the widest stride to the
// narrowest; where both have the same, at most a few places of one lie opposite
// a place of the other (more, or other strides: taken to meet if their spans
// do).
inline bool cells_meet(const CacheAxis* axes, int level, int count, int64_t size, int64_t apart) {
  int64_t keys = size, values = size, key_rest = size, value_rest = size;
  for (int i = count - 1; i >= level; --i) {
    key_rest = keys;
    value_rest = values;
    keys += (axes[i].count - 1) * axes[i].key;
    values += (axes[i].count - 1) * axes[i].value;
  }
  if (apart >= keys || -apart >= values) return false;
  if (level == count) return true;
  const CacheAxis& a = axes[level];
  if (a.key != a.value || a.key <= 0) return true;
  auto down = [](int64_t x, int64_t y) { return x / y - (x % y < 0 ? 1 : 0); };
  int64_t from = -down(value_rest - 1 + apart, a.key), to = down(key_rest - 1 - apart, a.key);
  from = from > 1 - a.count ? from : 1 - a.count;
  to = to < a.count - 1 ? to : a.count - 1;
  if (to - from > 2) return true;
  for (int64_t d = from; d <= to; ++d)
    if (cells_meet(axes, level + 1, count, size, apart + d * a.key)) return true;
  return false;
}

// Whether a cache's keys and values may share memory (which a call that writes
// both does not allow; interleaved ones do not share any).
inline bool keys_meet_values(const rkv_paged_cache* c) {
  const int64_t size = dtype_bytes(c->dtype);
  CacheAxis axes[4] = {{c->key_page_stride * size, c->value_page_stride * size, c->pages},
                       {c->key_head_stride * size, c->value_head_stride * size, c->heads},
                       {c->key_token_stride * size, c->value_token_stride * size, c->page_size},
                       {size, size, c->dim}};
  int count = 0;
  for (const CacheAxis& a : axes)
    if (a.count > 1) {
      int i = count++;
      const CacheAxis here = a;
      for (; i > 0 && axes[i - 1].key < here.key; --i) axes[i] = axes[i - 1];
      axes[i] = here;
    }
  return cells_meet(axes, 0, count, size,
                    static_cast<const char*>(c->values) - static_cast<const char*>(c->keys));
}

// The stride of an axis of `count` places; that of a single place is not read.
inline int64_t read_stride(int64_t stride, int64_t count) { return count > 1 ? stride : 0; }

// Whether (tokens, heads, dim) rows may lie among a cache's pages: the spans of
// both meet.
inline bool rows_meet_pages(const rkv_paged_cache* c, const void* rows, int64_t token_stride,
                            int64_t head_stride, int64_t tokens, int64_t heads) {
  const int64_t size = dtype_bytes(c->dtype);
  if (tokens <= 0 || heads <= 0) return false;
  const uint64_t from = reinterpret_cast<uint64_t>(rows);
  const uint64_t to = from + ((tokens - 1) * token_stride + (heads - 1) * head_stride + c->dim) * size;
  auto meets = [&](const void* pages, int64_t page, int64_t head, int64_t token) {
    const uint64_t first = reinterpret_cast<uint64_t>(pages);
    const uint64_t end = first + ((c->pages - 1) * page + (c->heads - 1) * head +
                                  (c->page_size - 1) * token + c->dim) * size;
    return from < end && first < to;
  };
  return meets(c->keys, c->key_page_stride, c->key_head_stride, c->key_token_stride) ||
         meets(c->values, c->value_page_stride, c->value_head_stride, c->value_token_stride);
}

}  // namespace rkv
