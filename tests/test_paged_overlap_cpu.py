"""Paged-cache calls whose tensors share memory: what would read or write a
place twice in one launch is refused, what lies apart is not."""

import ctypes

import pytest
import torch

from refinekv import PagedCache, Rotary, RotaryConfig, paged_append, paged_decode

F32 = torch.float32


def _tables(sequences=2, blocks=2):
    return (torch.arange(sequences * blocks, dtype=torch.int32).view(sequences, blocks),
            torch.tensor([3, 20], dtype=torch.int32)[:sequences].contiguous())


def _rows(cache):
    return torch.ones(cache.sequences, cache.heads, cache.head_dim)


def _c_append(cache, **over):
    """rkv_paged_append's code for tensors of these addresses (refused before
    any launch: nothing is followed here)."""
    from refinekv import _hip

    def strides(t):
        return (ctypes.c_int64 * 3)(*t.stride()[:3])

    view = _hip._PagedCache(
        keys=cache.keys.data_ptr(), key_strides=strides(cache.keys),
        values=cache.values.data_ptr(), value_strides=strides(cache.values),
        block_table=cache.block_table.data_ptr(), table_stride=cache.block_table.stride(0),
        lengths=cache.lengths.data_ptr(), pages=cache.pages, heads=cache.heads,
        page_size=cache.page_size, dim=cache.head_dim, sequences=cache.sequences,
        max_blocks=cache.max_blocks, dtype=_hip.DTYPE_CODES[cache.dtype])
    args = dict(rows=_rows(cache), query=0, q_heads=0, query_out=0, out_strides=(0, 0))
    args.update(over)
    dim, rows = cache.head_dim, args["rows"]
    code = _hip.lib().rkv_paged_append(
        ctypes.byref(view), args["query"], args["q_heads"] * dim, dim, args["q_heads"],
        args["query_out"], *args["out_strides"], rows.data_ptr(), rows.stride(0),
        rows.stride(1), rows.data_ptr(), rows.stride(0), rows.stride(1), cache.sequences, 0, 0, 0,
        0, 1.0, None)
    return code, _hip.lib().rkv_last_error().decode()


def _shared_caches():
    """(name, keys, values) whose cells overlap."""
    k = torch.zeros(4, 2, 16, 8)
    yield "one tensor", k, k
    pool = torch.zeros(9, 2, 16, 8)
    yield "a page on", pool[:8], pool[1:]
    flat = torch.zeros(5000)
    whole = torch.as_strided(flat, (4, 2, 16, 8), (256, 128, 8, 1))
    yield "half a row on", whole, torch.as_strided(flat, (4, 2, 16, 8), (256, 128, 8, 1), 4)
    yield "a row on", whole, torch.as_strided(flat, (4, 2, 16, 8), (256, 128, 8, 1), 8)
    yield "the other order", whole, torch.as_strided(flat, (4, 2, 16, 8), (256, 8, 16, 1))
    wide = torch.zeros(4, 2, 16, 12)
    yield "columns that meet", wide[..., :8], wide[..., 4:]


@pytest.mark.parametrize("name", [name for name, *_ in _shared_caches()])
def test_append_refuses_keys_and_values_that_share_memory(name):
    keys, values = {n: (k, v) for n, k, v in _shared_caches()}[name]
    cache = PagedCache(keys, values, *_tables())
    before = keys.clone()
    with pytest.raises(ValueError, match="share memory"):
        paged_append(_rows(cache), 2 * _rows(cache), cache)
    assert torch.equal(keys, before)
    code, why = _c_append(cache)
    assert code == 1 and "share memory" in why, (code, why)


def test_decode_over_shared_keys_and_values_still_answers():
    keys = torch.randn(4, 1, 16, 8, generator=torch.Generator().manual_seed(1))
    cache = PagedCache(keys, keys, *_tables())
    query = torch.zeros(2, 1, 8)
    want = torch.stack([keys[0, 0, :3].mean(0), torch.cat([keys[2, 0], keys[3, 0, :4]]).mean(0)])
    assert torch.allclose(paged_decode(query, cache)[:, 0], want, atol=1e-6)


def test_append_takes_interleaved_keys_and_values():
    """Keys and values in one tensor, by page, row, head or column, and caches
    one behind the other: every row is stored in its place."""
    both = torch.zeros(4, 2, 2, 16, 8)
    rows = torch.zeros(4, 16, 2, 2, 8)
    wide = torch.zeros(4, 2, 16, 16)
    flat = torch.zeros(4 * 512)
    layouts = {
        "pages": (both[:, 0], both[:, 1]), "heads": (both[:, :, 0], both[:, :, 1]),
        "rows": (rows[:, :, 0].transpose(1, 2), rows[:, :, 1].transpose(1, 2)),
        "columns": (wide[..., :8], wide[..., 8:]), "turned": (wide[..., 8:], wide[..., :8]),
        # a page's keys head by head, its values row by row behind them
        "orders": (torch.as_strided(flat, (4, 2, 16, 8), (512, 128, 8, 1)),
                   torch.as_strided(flat, (4, 2, 16, 8), (512, 8, 16, 1), 256)),
        "halves": (both.view(8, 2, 16, 8)[:4], both.view(8, 2, 16, 8)[4:]),
        "one page": (both[:1, 0], both[:1, 1]),
    }
    for name, (keys, values) in layouts.items():
        keys.zero_(), values.zero_()
        table, lengths = _tables()
        cache = PagedCache(keys, values, table, lengths)
        paged_append(_rows(cache), 2 * _rows(cache), cache)
        for t, fill in ((keys, 1.0), (values, 2.0)):
            want = torch.zeros(t.shape)
            want[0, :, 2] = fill
            if cache.pages > 3:
                want[3, :, 3] = fill
            assert torch.equal(t, want), name


def _cache(sequences=2):
    return PagedCache(torch.zeros(6, 2, 16, 8), torch.zeros(6, 2, 16, 8), *_tables(sequences))


def _places():
    """(cache, (2, 2, 8) rows in or beside it, whether in it)."""
    for name in ("keys", "values"):
        cache = _cache()
        pages = getattr(cache, name)
        yield cache, pages[5].transpose(0, 1)[:2], True
        yield cache, pages.view(-1)[-32:].view(2, 2, 8), True
        yield cache, pages.view(-1)[:32].view(2, 2, 8), True
    for place, inside in ((slice(0, 32), False), (slice(1, 33), True), (slice(-32, None), False),
                          (slice(-33, -1), True)):
        pool = torch.zeros(6 * 256 + 64)
        cache = _cache()
        cache = PagedCache(pool[32:-32].view(6, 2, 16, 8), cache.values, cache.block_table,
                           cache.lengths)
        yield cache, pool[place].view(2, 2, 8), inside


def test_append_refuses_queries_turned_into_the_cache():
    for cache, rows, inside in _places():
        args = dict(query=torch.ones(2, 2, 8), rotary=Rotary(RotaryConfig(head_dim=8)),
                    query_out=rows)
        if not inside:
            assert paged_append(_rows(cache), _rows(cache), cache, **args) is rows
            assert cache.keys.any()
            continue
        with pytest.raises(ValueError, match="overlaps the cache"):
            paged_append(_rows(cache), _rows(cache), cache, **args)
        assert not cache.keys.any() and not cache.values.any()
        code, why = _c_append(cache, query=4096, q_heads=2, query_out=rows.data_ptr(),
                              out_strides=rows.stride()[:2])
        assert code == 1 and "overlaps the cache" in why, (code, why)


def test_decode_refuses_an_output_in_the_cache():
    for cache, rows, inside in _places():
        if not rows.is_contiguous():
            continue
        query = torch.ones(2, 2, 8)
        if inside:
            with pytest.raises(ValueError, match="overlaps the cache"):
                paged_decode(query, cache, output=rows)
        else:
            assert paged_decode(query, cache, output=rows) is rows


def test_c_decode_refuses_an_output_in_the_cache():
    from refinekv import _hip

    page = 16 * 2 * 64 * 2  # bytes of a page's keys
    view = _hip._PagedCache(
        keys=1 << 20, values=1 << 21, block_table=4096, lengths=4096, pages=4, heads=2,
        page_size=16, dim=64, sequences=2, max_blocks=3, dtype=0, table_stride=3,
        key_strides=(ctypes.c_int64 * 3)(2048, 1024, 64),
        value_strides=(ctypes.c_int64 * 3)(2048, 1024, 64))
    out_bytes = 2 * 8 * 64 * 2
    for first in (1 << 20, 1 << 21):
        for out in (first, first + 4 * page - 16, first - out_bytes + 16):
            code = _hip.lib().rkv_paged_decode(ctypes.byref(view), 4096, 512, 64, 4, 0.125, out,
                                               4096, 0, None)
            assert code == 1 and b"overlaps the cache" in _hip.lib().rkv_last_error()
        for out in (first - out_bytes, first + 4 * page):  # (the workspace is too small)
            assert _hip.lib().rkv_paged_decode(ctypes.byref(view), 4096, 512, 64, 4, 0.125, out,
                                               4096, 0, None) == 4


def rows_of_pages(append):
    """append(cache, key, value, query, rotary) with rows that are views of
    pages the same call writes, against the same call with copies."""
    gen = torch.Generator().manual_seed(7)
    start = [torch.randn(6, 2, 16, 8, generator=gen) for _ in range(2)]
    rotary = Rotary(RotaryConfig(head_dim=8))
    results = []
    for copied in (False, True):
        cache = PagedCache(start[0].clone(), start[1].clone(), *_tables())
        # sequence 0's token goes to row 2 of page 0, sequence 1's to row 3 of page 3
        key = cache.keys[0].transpose(0, 1)[2:4]
        value = cache.keys[3].transpose(0, 1)[3:5]
        query = cache.values[0].transpose(0, 1)[1:3]
        if copied:
            key, value, query = key.clone(), value.clone(), query.clone()
        out = append(cache, key, value, query, rotary)
        results.append((out, cache.keys, cache.values))
    for got, want in zip(*results):
        assert torch.equal(got, want)
    assert not torch.equal(results[1][1], start[0])


def test_append_stores_what_its_rows_held_before():
    rows_of_pages(lambda cache, key, value, query, rotary: paged_append(
        key, value, cache, query=query, rotary=rotary))


def test_c_append_names_rows_in_the_cache():
    from refinekv import _hip

    for which in ("rows", "query"):
        cache = _cache()
        for name in ("keys", "values"):
            pages = getattr(cache, name)
            rows = pages[5].transpose(0, 1)[:2]
            over = (dict(rows=rows) if which == "rows" else
                    dict(query=rows.data_ptr(), q_heads=2, query_out=4096, out_strides=(16, 8)))
            code, why = _c_append(cache, **over)
            assert code == _hip.ROWS_IN_CACHE and "rows overlap the cache" in why, (code, why)
