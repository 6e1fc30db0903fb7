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

// The stride of an axis of `count` places; that of a single place is not read.
inline int64_t read_stride(int64_t stride, int64_t count) { return count > 1 ? stride : 0; }

}  // namespace rkv
