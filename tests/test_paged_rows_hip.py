"""Rows and outputs in unusual places, through the kernels (GPU)."""

import pytest
import torch

from refinekv import PagedCache, paged_append, paged_decode
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


def test_decode_into_an_output_at_any_address():
    """An output that starts anywhere its type may: the kernel stores whole
    vectors, so that the result goes there by a copy."""
    gen = torch.Generator().manual_seed(3)
    keys, values = (torch.randn(6, 2, 16, 64, generator=gen).to(torch.bfloat16).cuda()
                    for _ in range(2))
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    cache = PagedCache(keys, values, table,
                       torch.tensor([17, 40], dtype=torch.int32, device="cuda"))
    query = torch.randn(2, 6, 64, generator=gen).to(torch.bfloat16).cuda()
    want = paged_decode(query, cache, backend="hip")
    for first in (1, 4, 8):
        room = torch.full((query.numel() + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
        output = room[first:first + query.numel()].view(query.shape)
        for backend in ("auto", "hip"):
            output.zero_()
            assert paged_decode(query, cache, output=output, backend=backend) is output
            assert torch.equal(output, want)
        assert (room[:first] == 7).all() and (room[first + query.numel():] == 7).all()
    odd = keys.view(-1)[3:3 + query.numel()].view(query.shape)
    for backend in ("auto", "hip"):
        with pytest.raises(ValueError, match="overlaps the cache"):
            paged_decode(query, cache, output=odd, backend=backend)


def test_calls_that_cannot_be_captured_say_so():
    """What the kernels do not take goes to torch operations that read the
    lengths on the host: under a capture that is refused before any of them."""
    cache = PagedCache.empty(4, 1, 16, 64, 2, 2, dtype=torch.float32, device="cuda")
    wide = PagedCache.empty(4, 1, 16, 64, 2, 2, dtype=torch.float64, device="cuda")
    query = torch.zeros(2, 1, 64, device="cuda")
    paged_append(query, query, cache, backend="hip")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_append(query, query, cache, backend="hip")
        with pytest.raises(RuntimeError, match="cannot be captured.*bf16 or fp16"):
            paged_decode(query, cache)
        with pytest.raises(RuntimeError, match="cannot be captured.*backend='torch'"):
            paged_append(query, query, cache, backend="torch")
        with pytest.raises(RuntimeError, match="cannot be captured"):
            paged_append(query.new_zeros(0, 1, 64, dtype=torch.float64),
                         query.new_zeros(0, 1, 64, dtype=torch.float64), wide,
                         token_starts=cache.block_table.new_empty(3))
    graph.replay()
    torch.cuda.synchronize()
    assert not paged_decode(query, cache).any()


def test_decode_of_queries_with_far_heads():
    """Heads further apart than the kernel's 32-bit offsets reach are copied
    together, like rows that are not aligned."""
    gen = torch.Generator().manual_seed(4)
    keys, values = (torch.randn(4, 1, 16, 64, generator=gen).to(torch.bfloat16).cuda()
                    for _ in range(2))
    cache = PagedCache(keys, values, torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2),
                       torch.tensor([9, 30], dtype=torch.int32, device="cuda"))
    near = torch.randn(2, 2, 64, generator=gen).to(torch.bfloat16).cuda()
    far = torch.empty((1 << 25) + 1024, dtype=torch.bfloat16, device="cuda").as_strided(
        (2, 2, 64), (64, (1 << 25) + 8, 1)).copy_(near)
    want = paged_decode(near, cache, backend="hip")
    for backend in ("auto", "hip"):
        assert torch.equal(paged_decode(far, cache, backend=backend), want)
