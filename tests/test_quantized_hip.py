"""The paged cache in 4 bits and the decode's capped, biased and windowed
scores: the gfx950 kernels (GPU).

Appended bytes are compared with the torch restatement's, which the CPU tests
hold to the definition; decodes with the same in 64 bits.
"""

import math

import pytest
import torch

from paged_math import assert_within, pages_for
from quantized_math import attend64, decode64_quantized, quantize64
from refinekv import (PagedCache, QuantizedCache, Rotary, RotaryConfig, paged_append, paged_decode,
                      paged_read, quantized, rotate_heads)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    from refinekv import _hip

    _hip.lib()  # the HIP library must load: no fallback
    return _hip


def parts(cache):
    return cache.key_codes, cache.value_codes, cache.key_scales, cache.value_scales


def bits(t):
    return t.contiguous().view(torch.uint8)


def to(cache, device):
    """A copy on a device."""
    return QuantizedCache(*(t.to(device, copy=True) for t in (
        *parts(cache), cache.block_table, cache.lengths)), cache.dtype)


def filled(pages, heads, page, dim, table, lengths, dtype, gen):
    """A CPU cache whose pages hold what earlier calls left."""
    cache = QuantizedCache.empty(pages, heads, page, dim, len(lengths), len(table[0]), dtype=dtype)
    for t in (cache.key_codes, cache.value_codes):
        t.copy_(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
    for t in (cache.key_scales, cache.value_scales):
        t.copy_(torch.randint(0, 2000, t.shape, generator=gen) * 2.0 ** -10)
    cache.block_table.copy_(torch.tensor(table))
    cache.lengths.copy_(torch.tensor(lengths))
    return cache


# -- append and read ---------------------------------------------------------

def assert_turned(got, want, dtype):
    """Turned rows of two kernels, bf16 ones bit for bit.  In fp16 a product's
    sum and its rounding may be one instruction (rounded once) or two: the last
    bit may differ, 2^-10 of the value at most."""
    if dtype == BF16:
        assert torch.equal(bits(got), bits(want))
    else:
        assert bool(((got.double() - want.double()).abs()
                     <= 2.0 ** -10 * want.double().abs()).all())


def assert_same_caches(got, want):
    """Caches of rows turned by two kernels: bf16 ones bit for bit.  An fp16 key
    that differs by 2^-10 of it may fall to the next code (a scale), and a group
    whose bounds do have another scale (2^-6 of it, 15 times) and zero (2^-10)."""
    if got.dtype == BF16:
        for g, w in zip(parts(got), parts(want)):
            assert torch.equal(bits(g), bits(w))
        return
    (gk, gv, gs, gz), (wk, wv, ws, wz) = got.unpacked(), want.unpacked()
    assert torch.equal(gv, wv) and torch.equal(bits(gz), bits(wz))
    x, y = (quantized.dequantize(*t).double() for t in ((gk, gs), (wk, ws)))
    assert torch.equal(x.isnan(), y.isnan())
    room = 1.25 * ws[..., 0].double().repeat_interleave(32, -1) + 2.0 ** -9 * y.abs()
    live = ~y.isnan()
    assert bool(((x - y).abs() <= room)[live].all())
    assert int((gk != wk).sum()) <= 2 + wk.numel() // 1000


@pytest.mark.parametrize("dim,dtype,page,heads,q_heads", [
    (128, BF16, 16, 8, 32), (128, F16, 64, 4, 28), (64, BF16, 32, 1, 3), (32, F16, 16, 3, 3),
    (96, BF16, 16, 2, 2), (160, F16, 32, 1, 5), (192, BF16, 16, 2, 2), (224, F16, 16, 1, 1),
    (256, BF16, 128, 2, 16), (128, BF16, 256, 20, 20)])
def test_append_and_read(dim, dtype, page, heads, q_heads):
    gen = torch.Generator().manual_seed(dim + page)
    table = [[5, 1, -1], [2, 7, 4], [-1, -1, -1], [3, 9, 0], [6, -1, -1]]
    lengths = [page + 3, 2 * page + 1, 0, page + 2, 2]  # sequence 3: a page is not there
    new = [page + 3, 5, 0, 4, 3]                        # sequence 4: more rows than positions
    on_cpu = filled(9, heads, page, dim, table, lengths, dtype, gen)
    cache = to(on_cpu, DEV)
    starts = torch.tensor([0] + new).cumsum(0).int()
    tokens = int(starts[-1]) + 2
    key, value = (torch.randn(tokens, heads, dim, generator=gen).to(dtype) for _ in range(2))
    query = torch.randn(tokens, q_heads, dim, generator=gen).to(dtype)
    key[1, 0, 3], value[2, -1, dim - 1], value[0, 0, 0] = math.nan, math.inf, 5000.0
    key[3], value[3] = 0.25, 0.0
    paged_append(key, value, on_cpu, token_starts=starts)
    at = starts.to(DEV)
    assert paged_append(key.to(DEV), value.to(DEV), cache, token_starts=at,
                        backend="hip") is None
    for got, want in zip(parts(cache), parts(on_cpu)):
        assert torch.equal(bits(got.cpu()), bits(want))
    want = paged_read(on_cpu, tokens, token_starts=starts)
    got = paged_read(cache, tokens, token_starts=at, backend="hip")
    for g, w in zip(got, want):
        assert torch.equal(g.cpu().isnan(), w.isnan())
        assert torch.equal(g.cpu().nan_to_num(0), w.nan_to_num(0))
    # turned on the way: as turned before
    rotary = Rotary(RotaryConfig(head_dim=dim, base=500000.0), DEV)
    positions = [n - m + i for n, m in zip(lengths, new) for i in range(m)] + [0, 0]
    positions = torch.tensor(positions).clamp_min(0).to(DEV)
    q, k = rotate_heads(query.to(DEV), key.to(DEV), positions, rotary)
    again = to(cache, DEV)
    paged_append(k, value.to(DEV), again, token_starts=at)
    turned = paged_append(key.to(DEV), value.to(DEV), cache, query=query.to(DEV), rotary=rotary,
                          token_starts=at, backend="hip")
    assert_same_caches(cache, again)
    idle = int(starts[4])  # the row before its sequence's first position, and those of none
    live = [r for r in range(tokens - 2) if r != idle]
    assert_turned(turned[live], q[live], dtype)
    for r in (idle, tokens - 2, tokens - 1):
        assert torch.equal(bits(turned[r].cpu()), bits(query[r]))


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=64, rotary_dim=24), dict(head_dim=96, rotary_dim=36, interleaved=True),
    dict(head_dim=128, interleaved=True, scaling="yarn", factor=4.0),
    dict(head_dim=256, rotary_dim=64), dict(head_dim=64, rotary_dim=2), dict(head_dim=32),
    dict(head_dim=160, rotary_dim=80), dict(head_dim=128, scaling="llama3", factor=8.0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_turns(kwargs, dtype):
    """One token a sequence, parts of the head, either order of pairs: keys and
    queries as rotate_heads and an append without it."""
    config = RotaryConfig(base=1000000.0, **kwargs)
    dim, rotary = config.head_dim, Rotary(config, DEV)
    gen = torch.Generator().manual_seed(dim)
    lengths = [1, 37, 0, 64, 131072]
    cache = QuantizedCache.empty(6, 3, 64, dim, 5, 2048, dtype=dtype, device=DEV)
    cache.lengths.copy_(torch.tensor(lengths))
    cache.block_table[:, 0] = torch.arange(5)
    cache.block_table[4, 2047] = 5
    key, value = (torch.randn(5, 3, dim, generator=gen).to(dtype).to(DEV) for _ in range(2))
    query = torch.randn(5, 7, dim, generator=gen).to(dtype).to(DEV)
    positions = (cache.lengths - 1).clamp_min(0)
    q, k = rotate_heads(query, key, positions, rotary)
    other = to(cache, DEV)
    paged_append(k, value, other)
    turned = paged_append(key, value, cache, query=query, rotary=rotary, backend="hip")
    assert_same_caches(cache, other)
    live = [0, 1, 3, 4]
    assert_turned(turned[live], q[live], dtype)
    assert torch.equal(bits(turned[2]), bits(query[2]))


def test_append_views_in_place_and_unaligned():
    """Rows inside a fused projection, at odd addresses, in the other order;
    turned queries over the queries and at odd addresses."""
    gen = torch.Generator().manual_seed(3)
    rotary = Rotary(RotaryConfig(head_dim=64), DEV)
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    rows = torch.randn(50, 6, 64, generator=gen).to(BF16).to(DEV)
    caches = [QuantizedCache.empty(4, 1, 16, 64, 1, 4, device=DEV) for _ in range(4)]
    starts = torch.tensor([0, 50], dtype=torch.int32, device=DEV)
    results = []
    for i, cache in enumerate(caches):
        cache.block_table.copy_(table)
        cache.lengths.fill_(50)
        fused = rows.clone()
        if i == 1:  # heads, then tokens
            fused = fused.transpose(0, 1).contiguous().transpose(0, 1)
        if i == 2:  # two bytes off
            store = torch.empty(50 * 6 * 64 + 1, dtype=BF16, device=DEV)
            store[1:] = fused.reshape(-1)
            fused = store[1:].view(50, 6, 64)
        q, k, v = fused[:, :4], fused[:, 4:5], fused[:, 5:]
        out = q if i == 0 else torch.empty(50, 4, 72, dtype=BF16, device=DEV)[..., 4:68] if i == 3 \
            else None
        got = paged_append(k, v, cache, query=q, rotary=rotary, token_starts=starts, query_out=out,
                           backend="hip")
        assert out is None or got.data_ptr() == out.data_ptr()
        results.append((got.clone(), *parts(cache)))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("dtype,dim,layout", [(BF16, 128, "heads"), (F32, 36, "tokens"),
                                              (F16, 7, "heads"), (BF16, 6, "tokens")])
def test_read_of_a_16_bit_cache(dtype, dim, layout):
    gen = torch.Generator().manual_seed(5)
    keys, values = (torch.randn(7, 16, 3, dim, generator=gen).to(dtype).to(DEV)
                    for _ in range(2))
    if layout == "tokens":  # (pages, page, heads, dim) and its view
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    else:
        keys, values = (t.transpose(1, 2).contiguous() for t in (keys, values))
    table = torch.tensor([[2, 0], [3, -1], [6, 5]], dtype=torch.int32)
    lengths = torch.tensor([20, 18, 0], dtype=torch.int32)
    cache = PagedCache(keys, values, table.to(DEV), lengths.to(DEV))
    on_cpu = PagedCache(keys.cpu(), values.cpu(), table, lengths)
    for tokens, starts in ((3, None), (45, torch.tensor([0, 20, 38, 40], dtype=torch.int32))):
        want = paged_read(on_cpu, tokens, token_starts=starts)
        got = paged_read(cache, tokens, token_starts=None if starts is None else starts.to(DEV),
                         backend="hip")
        for g, w in zip(got, want):
            assert g.dtype == dtype and torch.equal(g.cpu().isnan(), w.isnan())
            assert torch.equal(g.cpu().nan_to_num(0), w.nan_to_num(0))
    assert paged_read(cache, 0, token_starts=torch.zeros(4, dtype=torch.int32, device=DEV),
                      backend="hip")[0].shape == (0, 3, dim)


# -- decode ------------------------------------------------------------------

def quantized_pages(lengths, page, heads, dim, dtype, gen, size=1.0, **kwargs):
    """(cache, (codes, scales, zeros) pairs in 64 bits): pages of randn, NaN in
    every row no sequence sees."""
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen, **kwargs)
    keys, values = keys * size, values * size
    plain = [quantized.quantize(t) for t in (keys, values)]
    cache = QuantizedCache.packed(plain[0][0], plain[1][0], plain[0][1], plain[1][1], table,
                                  torch.tensor(lengths, dtype=torch.int32), dtype=dtype)
    wide = [quantize64(t) for t in (keys, values)]
    return cache, [tuple(torch.from_numpy(w[i]) for w in wide) for i in range(3)]


SHAPES = [  # lengths, page, heads, group, dim, dtype
    ([1], 16, 1, 1, 64, BF16), ([1, 2, 3, 4, 5], 16, 1, 4, 128, BF16),
    ([0, 17, 0, 300, -2, 33], 16, 2, 4, 128, F16), ([31, 32, 33, 63, 64, 65], 32, 3, 7, 128, BF16),
    ([700, 1, 90], 64, 1, 16, 128, F16), ([250, 8], 16, 2, 5, 32, F16),
    ([100, 129], 128, 2, 3, 96, BF16), ([77, 200], 16, 1, 2, 160, F16),
    ([513], 256, 2, 8, 192, BF16), ([40, 41], 32, 1, 9, 224, F16), ([300, 7], 16, 2, 8, 256, BF16),
    ([2500], 32, 2, 4, 64, BF16), ([5000], 16, 1, 4, 128, BF16)]


@pytest.mark.parametrize("lengths,page,heads,group,dim,dtype", SHAPES)
def test_decode(lengths, page, heads, group, dim, dtype):
    gen = torch.Generator().manual_seed(dim + sum(lengths))
    on_cpu, wide = quantized_pages(lengths, page, heads, dim, dtype, gen)
    cache = to(on_cpu, DEV)
    query = torch.randn(len(lengths), heads * group, dim, generator=gen).to(dtype)
    got = paged_decode(query.to(DEV), cache, backend="hip")
    assert got.dtype == dtype
    want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, dim ** -0.5)
    assert_within(got, want, room)
    # capped, biased, windowed: windows that begin inside a tile, at one, before all
    slopes = torch.logspace(-3, 0, heads * group, base=2.0)
    for options in (dict(softcap=2.0), dict(window=19, softcap=30.0), dict(slopes=slopes),
                    dict(window=32), dict(window=1, slopes=slopes), dict(window=10 ** 9)):
        args = {k: v.to(DEV) if k == "slopes" else v for k, v in options.items()}
        got = paged_decode(query.to(DEV), cache, scaling=0.3, backend="hip", **args)
        want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, 0.3, **options)
        assert_within(got, want, room, str({k: v for k, v in options.items() if k != "slopes"}))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("key_size,query_size", [(1.0, 2.0 ** -40), (2.0 ** -7, 1.0),
                                                 (500.0, 0.002), (2.0 ** -12, 30.0)])
def test_decode_sizes(dtype, key_size, query_size):
    """Small and large keys and queries: codes times scales below fp16's normal
    numbers, queries far from 1."""
    if dtype == F16:
        query_size = max(query_size, 2.0 ** -10)
    gen = torch.Generator().manual_seed(11)
    lengths = [70, 150]
    on_cpu, wide = quantized_pages(lengths, 16, 2, 128, dtype, gen, size=key_size)
    query = (torch.randn(2, 8, 128, generator=gen) * query_size).to(dtype)
    query[0, 0] = query[0, 0] * 2.0 ** -8
    query[0, 0, 5] = 100 * query_size  # one large value: the others are small against it
    query[1, 3] = 0.0
    scaling = 1.0 / (key_size * query_size * 8)
    got = paged_decode(query.to(DEV), to(on_cpu, DEV), scaling=scaling, backend="hip")
    want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, scaling)
    assert_within(got, want, room)


def test_decode_bad_pages_and_windows_past_them():
    """A page outside the cache gives NaN where it is seen and nothing where
    the window has passed it; a length past the table gives NaN."""
    gen = torch.Generator().manual_seed(13)
    lengths = [100, 100, 49, 80]
    on_cpu, wide = quantized_pages(lengths, 16, 2, 64, BF16, gen)
    on_cpu.block_table[0, 1] = 1 << 20   # tokens 16..31
    on_cpu.block_table[1, 6] = -5        # tokens 96..99
    on_cpu.lengths[3] = 16 * on_cpu.max_blocks + 1
    lengths[3] = int(on_cpu.lengths[3])
    cache = to(on_cpu, DEV)
    query = torch.randn(4, 8, 64, generator=gen).to(BF16)
    for window, bad in ((0, [0, 1, 3]), (68, [1, 3]), (69, [0, 1, 3]), (4, [1, 3])):
        got = paged_decode(query.to(DEV), cache, window=window or None, backend="hip")
        assert [b for b in range(4) if bool(got[b].isnan().all())] == bad
        want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, 64 ** -0.5,
                                        window=window)
        assert_within(got, want, room, str(window))


def test_decode_nan_groups():
    """A NaN group of a key makes its sequence's head NaN; one of a value its
    dims; hidden by the window they do nothing."""
    gen = torch.Generator().manual_seed(17)
    lengths = [60]
    on_cpu, _ = quantized_pages(lengths, 16, 2, 128, BF16, gen)
    cache = to(on_cpu, DEV)
    query = torch.randn(1, 8, 128, generator=gen).to(BF16).to(DEV)
    clean = paged_decode(query, cache, backend="hip", window=20)
    row = torch.randn(1, 2, 128, generator=gen).to(BF16).to(DEV)
    key, value = row.clone(), row.clone()
    key[0, 0, 40] = math.nan
    value[0, 1, 70] = math.inf
    cache.lengths.fill_(36)  # token 35
    paged_append(key, value, cache)
    cache.lengths.fill_(60)
    got = paged_decode(query, cache, backend="hip")
    assert bool(got[0, :4].isnan().all())
    assert bool(got[0, 4:, 64:96].isnan().all())
    assert not bool(got[0, 4:, :64].isnan().any()) and not bool(got[0, 4:, 96:].isnan().any())
    assert torch.equal(bits(paged_decode(query, cache, backend="hip", window=20)), bits(clean))


@pytest.mark.parametrize("options", [dict(softcap=3.0), dict(window=100), dict(slopes=True),
                                     dict(window=33, softcap=50.0, slopes=True)])
@pytest.mark.parametrize("lengths,page,heads,group,dim,dtype", [
    ([40, 0, 333, 1], 16, 2, 4, 128, BF16), ([129, 2000], 64, 1, 7, 64, F16),
    ([64, 65], 32, 2, 1, 256, BF16), ([50], 16, 3, 16, 96, F16), ([95, 200], 128, 1, 3, 32, BF16)])
def test_scores_16_bits(lengths, page, heads, group, dim, dtype, options):
    gen = torch.Generator().manual_seed(dim)
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen)
    cache = PagedCache(*(t.to(DEV) for t in (keys, values, table)),
                       torch.tensor(lengths, dtype=torch.int32, device=DEV))
    query = torch.randn(len(lengths), heads * group, dim, generator=gen).to(dtype)
    slopes = torch.logspace(-3, 0, heads * group, base=2.0)
    args = {**options, **({"slopes": slopes.to(DEV)} if "slopes" in options else {})}
    got = paged_decode(query.to(DEV), cache, backend="hip", **args).cpu()
    for b, n in enumerate(lengths):
        for h in range(heads * group):
            if n == 0:
                assert not bool(got[b].any())
                continue
            k, v = (t[table[b, :-(-n // page)].long(), h // group].reshape(-1, dim)[:n]
                    for t in (keys, values))
            want, room = attend64(query[b, h:h + 1], k, v, torch.tensor([n - 1]), dim ** -0.5,
                                  dtype, options.get("softcap", 0.0),
                                  float(slopes[h]) if "slopes" in options else 0.0,
                                  options.get("window", 0))
            assert_within(got[b, h:h + 1], want, room, f"{b} {h}")


def test_window_past_bad_and_infinite_16_bits():
    """Pages behind the window may be gone, values behind it infinite or NaN."""
    gen = torch.Generator().manual_seed(19)
    keys, values, table = pages_for([100], 16, 2, 64, BF16, gen)
    args = [t.to(DEV) for t in (keys, values, table)]
    cache = PagedCache(*args, torch.tensor([100], dtype=torch.int32, device=DEV))
    query = torch.randn(1, 8, 64, generator=gen).to(BF16).to(DEV)
    clean = paged_decode(query, cache, window=30, backend="hip")
    page = int(table[0, 4])  # tokens 64..79; the window begins at 70
    cache.keys[page, :, :6] = math.nan
    cache.values[page, :, :3] = math.inf
    cache.values[page, :, 3:6] = math.nan
    cache.block_table[0, :4] = -1
    got = paged_decode(query, cache, window=30, backend="hip")
    assert torch.equal(bits(got), bits(clean))
    assert bool(paged_decode(query, cache, window=40, backend="hip").isnan().all())
    # without options: the call as it was
    whole = paged_decode(query, cache, window=30, softcap=1e30, backend="hip")
    assert_within(whole, clean.cpu().double(), clean.cpu().double().abs() * 2.0 ** -6 + 1e-3)


def test_streams_graphs_and_workspace():
    """A step captured once and replayed as lengths grow, beside eager calls of
    another shape on the same workspace; a call on another stream."""
    gen = torch.Generator().manual_seed(23)
    cache = QuantizedCache.empty(20, 2, 16, 128, 3, 6, device=DEV)
    cache.block_table.copy_(torch.randperm(20, generator=gen)[:18].view(3, 6))
    cache.lengths.copy_(torch.tensor([30, 0, 61]))
    starts = torch.tensor([0, 30, 30, 91], dtype=torch.int32, device=DEV)
    rows = [torch.randn(91, 2, 128, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    paged_append(*rows, cache, token_starts=starts)
    rotary = Rotary(RotaryConfig(head_dim=128), DEV)
    slopes = torch.linspace(0.1, 0.4, 8, device=DEV)
    key, value = (torch.randn(3, 2, 128, device=DEV, dtype=BF16) for _ in range(2))
    query = torch.randn(3, 8, 128, device=DEV, dtype=BF16)
    active = torch.tensor([1, 0, 1], dtype=torch.int32, device=DEV)
    workspace = {}

    def step():
        cache.lengths.add_(active)
        q = paged_append(key, value, cache, query=query, rotary=rotary)
        return paged_decode(q, cache, workspace=workspace, softcap=30.0, slopes=slopes, window=50)

    def eager(lengths):
        other = to(cache, DEV)
        other.lengths.copy_(lengths)
        q = paged_append(key, value, other, query=query, rotary=rotary)
        return paged_decode(q, other, softcap=30.0, slopes=slopes, window=50)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        key.normal_()
        value.normal_()
        query.normal_()
        lengths = cache.lengths + active
        want = eager(lengths)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.lengths, lengths)
        assert torch.equal(bits(out), bits(want)), i
        paged_decode(query[:, :4].contiguous(), cache, workspace=workspace)
    assert not bool(out[1].any())


def test_offsets_past_32_bits():
    """Pages whose codes lie more than 2^32 bytes into the cache."""
    pages = 40000  # 16 heads x 256 tokens x 64 bytes: 10.5 GB of codes a side
    gen = torch.Generator().manual_seed(29)
    shape = (pages, 16, 256)
    cache = QuantizedCache(*(torch.empty(*shape, 64, dtype=torch.uint8, device=DEV)
                             for _ in range(2)),
                           *(torch.empty(*shape, 4, 2, dtype=F16, device=DEV) for _ in range(2)),
                           torch.tensor([[pages - 1, 3], [20001, pages - 2]], dtype=torch.int32,
                                        device=DEV),
                           torch.tensor([300, 512], dtype=torch.int32, device=DEV))
    small = QuantizedCache.empty(4, 16, 256, 128, 2, 2, device=DEV)
    small.block_table.copy_(torch.tensor([[0, 1], [2, 3]]))
    small.lengths.copy_(cache.lengths)
    rows = [torch.randn(812, 16, 128, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    starts = torch.tensor([0, 300, 812], dtype=torch.int32, device=DEV)
    query = torch.randn(2, 64, 128, generator=gen).to(BF16).to(DEV)
    results = []
    for c in (cache, small):
        paged_append(*rows, c, token_starts=starts)
        results.append((*paged_read(c, 812, token_starts=starts), paged_decode(query, c)))
    for a, b in zip(*results):
        assert torch.equal(bits(a), bits(b))


def test_refusals():
    cache = QuantizedCache.empty(4, 2, 16, 64, 3, 2, device=DEV)
    query = torch.zeros(3, 4, 64, dtype=BF16, device=DEV)
    with pytest.raises(ValueError):
        paged_decode(query, cache, slopes=torch.zeros(4))  # another device
    with pytest.raises(ValueError):
        paged_decode(query, cache, output=query)
    pool = cache.key_codes.view(-1).view(BF16)
    with pytest.raises(ValueError):
        paged_decode(query, cache, output=pool[:768].view(3, 4, 64))
    big = torch.zeros(3, 34, 64, dtype=BF16, device=DEV)
    with pytest.raises(TypeError):
        paged_decode(big, cache, backend="hip")
    assert not bool(paged_decode(big, cache).any())  # torch operations answer
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(graph):
            paged_decode(big, cache)
    raw = torch.zeros(2 * 16 * 32 * 4 + 8, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):  # codes at an odd address
        QuantizedCache(raw[8:].view(4, 2, 16, 32), cache.value_codes, cache.key_scales,
                       cache.value_scales, cache.block_table, cache.lengths)


def test_scales_of_nothing():
    """A scale of 0, one that vanishes against a zero query's, negative ones."""
    gen = torch.Generator().manual_seed(31)
    lengths = [40, 17, 0]
    on_cpu, wide = quantized_pages(lengths, 16, 1, 64, BF16, gen)
    query = torch.randn(3, 4, 64, generator=gen).to(BF16)
    query[0, 1] = 0.0
    for scaling in (0.0, 1e-20, -0.2):
        got = paged_decode(query.to(DEV), to(on_cpu, DEV), scaling=scaling, backend="hip")
        want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, scaling)
        assert_within(got, want, room, str(scaling))


def test_query_out_among_the_pages():
    """Refused, at an odd address as well (where a copy would be made first)."""
    cache = QuantizedCache.empty(64, 1, 16, 64, 2, 2, device=DEV)
    rows = torch.zeros(2, 1, 64, dtype=BF16, device=DEV)
    rotary = Rotary(RotaryConfig(head_dim=64), DEV)
    pool = cache.value_codes.view(-1).view(BF16)
    for first in (0, 1):
        with pytest.raises(ValueError):
            paged_append(rows, rows, cache, query=rows, rotary=rotary,
                         query_out=pool[first:first + 128].view(2, 1, 64))


@pytest.mark.parametrize("scores", [{}, dict(softcap=20.0)])
@pytest.mark.parametrize("four", [True, False])
def test_widest_group_and_head(four, scores):
    """The most LDS that a workgroup's parts take: 16 query heads of 256 dims, rows
    that several waves and workgroups hold parts of."""
    gen = torch.Generator().manual_seed(37)
    lengths = [700, 3, 41000]
    query = torch.randn(3, 16, 256, generator=gen).to(BF16)
    if four:
        on_cpu, wide = quantized_pages(lengths, 64, 1, 256, BF16, gen)
        got = paged_decode(query.to(DEV), to(on_cpu, DEV), backend="hip", **scores)
        want, room = decode64_quantized(query, *wide, on_cpu.block_table, lengths, 1 / 16, **scores)
        assert_within(got, want, room)
        return
    keys, values, table = pages_for(lengths, 64, 1, 256, BF16, gen)
    cache = PagedCache(*(t.to(DEV) for t in (keys, values, table)),
                       torch.tensor(lengths, dtype=torch.int32, device=DEV))
    got = paged_decode(query.to(DEV), cache, backend="hip", **scores).cpu()
    for b, n in enumerate(lengths):
        k, v = (t[table[b, :-(-n // 64)].long(), 0].reshape(-1, 256)[:n] for t in (keys, values))
        want, room = attend64(query[b], k, v, torch.full((16,), n - 1), 1 / 16, BF16,
                              scores.get("softcap", 0.0))
        assert_within(got[b], want, room, str(b))


def test_rows_in_the_cache_are_refused():
    cache = QuantizedCache.empty(16, 2, 16, 64, 3, 2, device=DEV)
    inside = cache.value_codes.view(-1).view(BF16)[:384].view(3, 2, 64)
    rows = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    for change in (dict(key=inside), dict(value=inside)):
        with pytest.raises(ValueError, match="overlap the cache"):
            paged_append(**{**dict(key=rows, value=rows, cache=cache, backend="hip"), **change})
