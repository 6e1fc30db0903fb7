"""Rows that are views of the cache's own pages, through the kernels (GPU)."""

import pytest
import torch

from refinekv import PagedCache, paged_append
from test_paged_overlap_cpu import rows_of_pages

pytestmark = pytest.mark.gpu


def test_append_stores_what_its_rows_held_before():
    def append(cache, key, value, query, rotary):
        there = PagedCache(*(getattr(cache, n).cuda()
                             for n in ("keys", "values", "block_table", "lengths")))

        def same(t):  # the view on the GPU
            for n in ("keys", "values"):
                if t.untyped_storage().data_ptr() == getattr(cache, n).untyped_storage().data_ptr():
                    return getattr(there, n).as_strided(t.shape, t.stride(), t.storage_offset())
            return t.cuda()

        turns = type(rotary)(rotary.config, "cuda")
        out = paged_append(same(key), same(value), there, query=same(query), rotary=turns,
                           backend="hip")
        cache.keys.copy_(there.keys), cache.values.copy_(there.values)
        return out.cpu()

    rows_of_pages(append)
