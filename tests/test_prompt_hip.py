"""Prompts' attention: the gfx950 kernels against the same in 64 bits (GPU)."""

import math

import pytest
import torch

from paged_math import pages_for
from prompt_math import assert_rows, prompt64
from refinekv import (PagedCache, QuantizedCache, Rotary, RotaryConfig, paged_append, paged_decode,
                      paged_prompt, paged_read, prompt_attention, rotate_heads)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    from refinekv import _hip

    _hip.lib()  # the HIP library must load: no fallback
    return _hip


def bits(t):
    return t.contiguous().view(torch.uint8)


def on_gpu(options):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in options.items()}


def ragged(counts, heads, group, dim, dtype, gen, behind=3):
    tokens = sum(counts) + behind
    starts = torch.tensor([0] + list(counts)).cumsum(0).int()
    rows = [torch.randn(tokens, n, dim, generator=gen).to(dtype)
            for n in (heads * group, heads, heads)]
    return starts, *rows


def options_for(counts, q_heads):
    slopes = torch.logspace(-4, 0, q_heads, base=2.0)
    prefix = torch.tensor([max(n // 3, 0) * (b % 3) - b % 2 for b, n in enumerate(counts)]).int()
    return [{}, dict(window=1), dict(window=70), dict(softcap=2.0), dict(slopes=slopes),
            dict(prefix=prefix), dict(prefix=prefix, window=33, softcap=20.0, slopes=slopes),
            dict(scaling=-0.3), dict(scaling=0.0)]


SHAPES = [  # rows, heads, group, dim, dtype
    ([1], 1, 1, 64, BF16), ([1, 2, 3], 2, 4, 128, BF16), ([37], 8, 4, 128, BF16),
    ([0, 31, 0, 32, 33, 0], 1, 1, 128, F16), ([63, 64, 65], 2, 1, 128, BF16),
    ([130, 5], 1, 7, 128, F16), ([300], 1, 16, 64, BF16), ([129, 127], 2, 3, 32, F16),
    ([70, 200], 1, 2, 96, BF16), ([90], 2, 5, 160, F16), ([33, 100], 1, 8, 192, BF16),
    ([65], 1, 4, 224, F16), ([40, 1, 97], 2, 2, 256, BF16), ([600], 1, 2, 64, F16),
    ([20], 1, 40, 128, BF16)]


@pytest.mark.parametrize("counts,heads,group,dim,dtype", SHAPES)
def test_rows(counts, heads, group, dim, dtype):
    gen = torch.Generator().manual_seed(dim + sum(counts))
    starts, query, key, value = ragged(counts, heads, group, dim, dtype, gen)
    rows = [t.to(DEV) for t in (query, key, value)]
    for options in options_for(counts, heads * group):
        what = str({k: v for k, v in options.items() if not isinstance(v, torch.Tensor)})
        got = prompt_attention(*rows, token_starts=starts.to(DEV), backend="hip",
                               **on_gpu(options))
        want, room = prompt64(query, key, value, starts, starts, **options)
        assert_rows(got, want, room, what)
        kept = torch.full_like(rows[0], 7.0)
        prompt_attention(*rows, token_starts=starts.to(DEV), backend="hip", output=kept,
                         **on_gpu(options))
        end = int(starts[-1])
        assert torch.equal(bits(kept[:end]), bits(got[:end])), what
        assert bool((kept[end:] == 7.0).all()) and not bool(got[end:].any())


@pytest.mark.parametrize("n,heads,group,dim,dtype", [(1500, 2, 2, 128, BF16), (1111, 1, 3, 64, F16)])
def test_one_long_sequence(n, heads, group, dim, dtype):
    gen = torch.Generator().manual_seed(n)
    _, query, key, value = ragged([n], heads, group, dim, dtype, gen, behind=0)
    key[::97] = (key[::97] * 4).to(dtype)  # peaks, late maxima
    ends = torch.tensor([0, n])
    for options in ({}, dict(window=500), dict(softcap=10.0)):
        got = prompt_attention(*(t.to(DEV) for t in (query, key, value)), backend="hip", **options)
        want, room = prompt64(query, key, value, ends, ends, **options)
        assert_rows(got, want, room, str(options))


@pytest.mark.parametrize("new,keys,group,dim,dtype", [
    ([5], [3000], 4, 128, BF16), ([1, 40], [2500, 700], 7, 64, F16), ([17, 0, 3], [900, 5, 0], 1,
                                                                      256, BF16),
    ([30], [20], 2, 128, F16), ([9], [5000], 3, 96, BF16)])
def test_few_rows_over_many_keys(new, keys, group, dim, dtype):
    """Calls that share their keys out and join the shares; more rows than
    keys."""
    gen = torch.Generator().manual_seed(sum(keys))
    starts, query, _, _ = ragged(new, 2, group, dim, dtype, gen)
    key_starts, _, key, value = ragged(keys, 2, 1, dim, dtype, gen)
    slopes = torch.logspace(-9, -2, 2 * group, base=2.0)
    workspace = {}
    for options in ({}, dict(window=300, softcap=5.0), dict(slopes=slopes),
                    dict(prefix=torch.tensor([k // 2 for k in keys]).int(), window=2000)):
        want, room = prompt64(query, key, value, starts, key_starts, **options)
        for w in (None, workspace):
            got = prompt_attention(*(t.to(DEV) for t in (query, key, value)),
                                   token_starts=starts.to(DEV), key_starts=key_starts.to(DEV),
                                   workspace=w, backend="hip", **on_gpu(options))
            assert_rows(got, want, room, str([k for k in options]))
    assert workspace if max(keys) > 512 else not workspace


@pytest.mark.parametrize("page,heads,group,dim,dtype,layout", [
    (16, 2, 4, 128, BF16, "heads"), (32, 1, 7, 64, F16, "tokens"), (64, 2, 1, 96, BF16, "heads"),
    (256, 1, 3, 256, F16, "heads"), (128, 3, 2, 32, BF16, "tokens"), (16, 1, 5, 192, BF16, "heads")])
def test_pages(page, heads, group, dim, dtype, layout):
    """Chunks over pages as prompt_attention over the rows the pages hold."""
    gen = torch.Generator().manual_seed(page + dim)
    lengths, new = [70, 0, 333, 1, 129, 40], [70, 0, 50, 1, 128, 1]
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen)
    if layout == "tokens":
        keys, values = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (keys, values))
    cache = PagedCache(*(t.to(DEV) for t in (keys, values, table)),
                       torch.tensor(lengths, dtype=torch.int32, device=DEV))
    starts, query, _, _ = ragged(new, heads, group, dim, dtype, gen)
    ends = torch.tensor([0] + lengths).cumsum(0).int()
    key, value = paged_read(cache, int(ends[-1]), token_starts=ends.to(DEV))
    for options in options_for(lengths, heads * group):
        got = paged_prompt(query.to(DEV), cache, token_starts=starts.to(DEV), backend="hip",
                           **on_gpu(options))
        want, room = prompt64(query, key.cpu(), value.cpu(), starts, ends, **options)
        assert_rows(got, want, room, str([k for k in options]))
    # one token a sequence, as the decode
    one = paged_prompt(query[:6].to(DEV), cache, backend="hip", window=90)
    want, room = prompt64(query[:6], key.cpu(), value.cpu(), [0, 1, 2, 3, 4, 5, 6], ends, window=90)
    assert_rows(one, want, room)


def test_pages_that_are_not_there():
    gen = torch.Generator().manual_seed(5)
    lengths, new = [100, 200, 64, 50], [40, 200, 5, 50]
    keys, values, table = pages_for(lengths, 16, 2, 64, BF16, gen)
    clean = PagedCache(*(t.to(DEV) for t in (keys, values, table)),
                       torch.tensor(lengths, dtype=torch.int32, device=DEV))
    table = table.clone()
    table[0, 1] = -9          # tokens 16..31: seen by all
    table[1, 7] = 1 << 30     # tokens 112..127: seen from row 112 on
    cache = PagedCache(clean.keys, clean.values, table.to(DEV), clean.lengths.clone())
    cache.lengths[2] = 16 * cache.max_blocks + 1
    starts = torch.tensor([0] + new).cumsum(0).int().to(DEV)
    query = torch.randn(295, 4, 64, generator=gen).to(BF16).to(DEV)
    want = paged_prompt(query, clean, token_starts=starts, backend="hip")
    got = paged_prompt(query, cache, token_starts=starts, backend="hip")
    nan = torch.zeros(295, dtype=torch.bool)
    nan[:40] = nan[152:240] = nan[240:245] = True
    assert torch.equal(got.isnan().all(2).all(1).cpu(), nan)
    assert torch.equal(bits(got[~nan.to(DEV)]), bits(want[~nan.to(DEV)]))
    # a window that has passed them
    got = paged_prompt(query, cache, token_starts=starts, window=28, backend="hip")
    want = paged_prompt(query, clean, token_starts=starts, window=28, backend="hip")
    nan[:] = False
    nan[240:245] = True
    nan[152:152 + 16 + 27] = True  # rows 112 .. 127 + 27 see the second
    assert torch.equal(got.isnan().all(2).all(1).cpu(), nan)
    assert torch.equal(bits(got[~nan.to(DEV)]), bits(want[~nan.to(DEV)]))


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (160, BF16)])
def test_infinities_and_nan(dim, dtype):
    """Infinite and NaN keys and values reach the rows that see them alone."""
    gen = torch.Generator().manual_seed(dim)
    counts = [150, 70]
    starts, query, key, value = ragged(counts, 1, 2, dim, dtype, gen, behind=1)
    value[40, 0, 3], value[90, 0, 4], value[100, 0, 3] = math.inf, math.nan, -math.inf
    value[149, 0, :] = -math.inf
    value[200, 0, dim - 1] = math.inf
    key[215, 0, 5] = math.nan
    value[220] = math.nan  # of no sequence
    for options in ({}, dict(window=30), dict(prefix=torch.tensor([50, 0]).int())):
        got = prompt_attention(*(t.to(DEV) for t in (query, key, value)),
                               token_starts=starts.to(DEV), backend="hip", **on_gpu(options))
        want, room = prompt64(query, key, value, starts, starts, **options)
        assert_rows(got, want, room, str([k for k in options]))


def test_views_and_outputs():
    """Rows inside a fused projection, at odd addresses, in the other order;
    an output at an odd address."""
    gen = torch.Generator().manual_seed(7)
    fused = torch.randn(77, 8, 64, generator=gen).to(BF16).to(DEV)
    starts = torch.tensor([0, 30, 77], dtype=torch.int32, device=DEV)
    parts = [t.contiguous() for t in (fused[:, :4], fused[:, 4:6], fused[:, 6:])]
    want = prompt_attention(*parts, token_starts=starts, backend="hip")
    odd = torch.empty(77 * 8 * 64 + 1, dtype=BF16, device=DEV)
    odd[1:] = fused.reshape(-1)
    for rows in (fused, odd[1:].view(77, 8, 64),
                 fused.transpose(0, 1).contiguous().transpose(0, 1)):
        got = prompt_attention(rows[:, :4], rows[:, 4:6], rows[:, 6:], token_starts=starts,
                               backend="hip")
        assert torch.equal(bits(got), bits(want))
    out = torch.empty(77 * 4 * 64 + 1, dtype=BF16, device=DEV)[1:].view(77, 4, 64)
    assert prompt_attention(*parts, token_starts=starts, output=out,
                            backend="hip").data_ptr() == out.data_ptr()
    assert torch.equal(bits(out), bits(want))
    empty = prompt_attention(*(t[:0] for t in parts), backend="hip")
    assert empty.shape == (0, 4, 64)
    none = prompt_attention(parts[0], parts[1][:0], parts[2][:0], token_starts=starts,
                            key_starts=torch.zeros_like(starts), backend="hip")
    assert not bool(none.any())


def test_starts_that_are_no_starts():
    """Device starts the host cannot check stay inside the rows."""
    gen = torch.Generator().manual_seed(8)
    _, query, key, value = ragged([50], 1, 2, 64, BF16, gen, behind=0)
    rows = [t.to(DEV) for t in (query, key, value)]
    for starts in ([0, 1 << 30], [-5, 20], [40, 10], [60, 70], [-(2 ** 31), 2 ** 31 - 1]):
        at = torch.tensor(starts, dtype=torch.int32, device=DEV)
        first = min(max(starts[0], 0), 50)
        end = min(max(starts[1], first), 50)
        got = prompt_attention(*rows, token_starts=at, backend="hip")
        want, room = prompt64(query, key, value, [first, end], [first, end])
        assert_rows(got, want, room, str(starts))


def test_graph_and_streams():
    """A layer's chunk (turn, append, attend) captured once and replayed as the
    sequences grow, with eager calls between; the same on another stream."""
    gen = torch.Generator().manual_seed(9)
    cache = PagedCache.empty(40, 2, 16, 64, 2, 20, device=DEV)
    cache.block_table.copy_(torch.randperm(40, generator=gen).view(2, 20))
    starts = torch.tensor([0, 7, 12], dtype=torch.int32, device=DEV)
    grow = torch.tensor([7, 5], dtype=torch.int32, device=DEV)
    rotary = Rotary(RotaryConfig(head_dim=64), DEV)
    query, key, value = (torch.randn(12, n, 64, device=DEV, dtype=BF16) for n in (4, 2, 2))
    workspace = {}

    def chunk(cache, workspace):
        cache.lengths.add_(grow)
        q = paged_append(key, value, cache, query=query, rotary=rotary, token_starts=starts)
        return paged_prompt(q, cache, token_starts=starts, window=40, workspace=workspace,
                            backend="hip")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chunk(cache, workspace)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chunk(cache, workspace)
    for i in range(4):
        for t in (query, key, value):
            t.normal_()
        other = PagedCache(cache.keys.clone(), cache.values.clone(), cache.block_table,
                           cache.lengths.clone())
        want = chunk(other, None)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(want)), i
        assert torch.equal(bits(cache.keys), bits(other.keys))
        paged_prompt(query[:2], cache, workspace=workspace)


def test_serving_in_4_bits():
    """The operators together: prompts turned, attended over their own rows and
    appended in 4 bits, a chunk over rows read back, decode steps; against the
    torch operations on the CPU."""
    gen = torch.Generator().manual_seed(10)
    rotary = [Rotary(RotaryConfig(head_dim=64), d) for d in (DEV, "cpu")]
    caches = [QuantizedCache.empty(12, 2, 16, 64, 2, 6, device=d) for d in (DEV, "cpu")]
    table = torch.randperm(12, generator=gen).view(2, 6).int()
    prompts, chunk = [50, 23], [9, 14]
    results = [[], []]
    draws = [[torch.randn(n, h, 64, generator=gen).to(BF16) for h in (6, 2, 2)]
             for n in (sum(prompts), sum(chunk), 2, 2)]
    for cache, turn, found in zip(caches, rotary, results):
        dev = cache.device
        cache.block_table.copy_(table)
        q, k, v = (t.to(dev) for t in draws[0])
        starts = torch.tensor([0] + prompts).cumsum(0).int().to(dev)
        cache.lengths.copy_(torch.tensor(prompts))
        at = torch.cat([torch.arange(n) for n in prompts]).to(dev)
        q, k = rotate_heads(q, k, at, turn)
        found.append(prompt_attention(q, k, v, token_starts=starts))
        paged_append(k, v, cache, token_starts=starts)
        q, k, v = (t.to(dev) for t in draws[1])
        new = torch.tensor([0] + chunk).cumsum(0).int().to(dev)
        cache.lengths.add_(torch.tensor(chunk, device=dev))
        q = paged_append(k, v, cache, query=q, rotary=turn, token_starts=new)
        total = [a + b for a, b in zip(prompts, chunk)]
        ends = torch.tensor([0] + total).cumsum(0).int().to(dev)
        k, v = paged_read(cache, sum(total), token_starts=ends)
        found.append(prompt_attention(q, k, v, token_starts=new, key_starts=ends, softcap=30.0))
        for q, k, v in draws[2:]:
            cache.lengths.add_(1)
            q = paged_append(k.to(dev), v.to(dev), cache, query=q.to(dev), rotary=turn)
            found.append(paged_decode(q, cache, softcap=30.0))
    for got, want in zip(*results):
        # weights of bf16 on both sides' 32-bit sums, outputs rounded: 2^-8 each
        assert float((got.cpu().float() - want.float()).abs().max()) <= 3 * 2.0 ** -8 * float(
            want.float().abs().max())


def test_refusals():
    q, k = torch.zeros(6, 4, 32, dtype=BF16, device=DEV), torch.zeros(6, 2, 32, dtype=BF16,
                                                                      device=DEV)
    with pytest.raises(ValueError):
        prompt_attention(q, k, k.clone(), token_starts=torch.tensor([0, 6]).int())  # on the CPU
    wide = torch.zeros(6, 4, 40, dtype=BF16, device=DEV)
    with pytest.raises(TypeError):
        prompt_attention(wide, wide, wide.clone(), backend="hip")
    assert not bool(prompt_attention(wide, wide, wide.clone()).any())  # torch operations answer
    cache = QuantizedCache.empty(4, 2, 16, 32, 6, 2, device=DEV)
    with pytest.raises(TypeError):
        paged_prompt(q, cache, backend="hip")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(graph):
            paged_prompt(q, cache)


def test_starts_that_overlap():
    """Several sequences whose device starts overlap ask for more tiles than the
    rows have: whatever is written lies inside, and later calls are right."""
    gen = torch.Generator().manual_seed(12)
    _, query, key, value = ragged([40], 1, 2, 64, BF16, gen, behind=0)
    rows = [t.to(DEV) for t in (query, key, value)]
    many = torch.tensor([0, 40] * 33, dtype=torch.int32, device=DEV)
    far = torch.tensor([0, 2 ** 31 - 1] * 33, dtype=torch.int32, device=DEV)
    long_keys = [torch.randn(4000, 1, 64, generator=gen).to(BF16).to(DEV) for _ in range(2)]
    workspace = {}
    for starts in (many, far):
        guard = torch.full((42, 2, 64), 7.0, dtype=BF16, device=DEV)
        prompt_attention(*rows, token_starts=starts, output=guard[1:41], backend="hip")
        prompt_attention(rows[0], *long_keys, token_starts=starts,
                         key_starts=torch.tensor([0, 4000] * 33, dtype=torch.int32, device=DEV),
                         output=guard[1:41], workspace=workspace, backend="hip")
        assert bool((guard[0] == 7.0).all()) and bool((guard[41] == 7.0).all())
    ends = torch.tensor([0, 40])
    got = prompt_attention(*rows, backend="hip")
    want, room = prompt64(query, key, value, ends, ends)
    assert_rows(got, want, room)


@pytest.mark.parametrize("dim,group,dtype", [(64, 1, BF16), (128, 3, F16)])
def test_slopes_of_all_sizes(dim, group, dtype):
    """Slopes below zero, of nothing and too large for a shared bias; scales that
    are too small or large for one, or 1; caps beside them."""
    gen = torch.Generator().manual_seed(dim)
    counts = (300, 65)
    starts, query, key, value = ragged(counts, 2, group, dim, dtype, gen)
    rows = [t.to(DEV) for t in (query, key, value)]
    slopes = torch.logspace(-9, 0, 2 * group, base=2.0)
    prefix = torch.tensor([130, 3]).int()
    one = math.log(2.0)  # (times log2 e: about 1)
    mixed = slopes.clone()
    mixed[0] = 1e25
    for options in (dict(slopes=-slopes), dict(slopes=slopes * 0), dict(slopes=mixed),
                    dict(slopes=slopes, scaling=2.0 ** -24), dict(slopes=slopes, scaling=-0.1),
                    dict(slopes=slopes, scaling=one), dict(softcap=3.0, scaling=one),
                    dict(slopes=-slopes, softcap=3.0, window=100),
                    dict(slopes=slopes, prefix=prefix, window=70)):
        got = prompt_attention(*rows, token_starts=starts.to(DEV), backend="hip",
                               **on_gpu(options))
        want, room = prompt64(query, key, value, starts, starts, **options)
        what = str({k: v if isinstance(v, float) else str(v) for k, v in options.items()})
        assert_rows(got, want, room, what)


@pytest.mark.parametrize("before,behind", [(0, 9001), (1300, 700), (5000, 4000)])
def test_rows_of_no_sequence(before, behind):
    """A padded batch: zeros in a new tensor, left alone in `output`."""
    gen = torch.Generator().manual_seed(before)
    counts, heads, group, dim = (50, 0, 33), 3, 2, 64
    _, query, key, value = ragged(counts, heads, group, dim, F16, gen, behind=before + behind)
    starts = torch.tensor([before, before + 50, before + 50, before + 83]).int()
    rows = [t.to(DEV) for t in (query, key, value)]
    poison = torch.full_like(rows[0], 7.0)  # (memory that the new tensor may take)
    del poison
    got = prompt_attention(*rows, token_starts=starts.to(DEV), backend="hip")
    want, room = prompt64(query, key, value, starts, starts)
    assert_rows(got, want, room, "padded")
    assert not bool(got[:before].any()) and not bool(got[before + 83:].any())
    kept = torch.full_like(rows[0], 7.0)
    prompt_attention(*rows, token_starts=starts.to(DEV), backend="hip", output=kept)
    inside = slice(before, before + 83)
    assert torch.equal(bits(kept[inside]), bits(got[inside]))
    assert bool((kept[:before] == 7.0).all()) and bool((kept[before + 83:] == 7.0).all())


def test_more_sequences_than_lanes():
    """More sequences than a wave has lanes, most of them empty or of a row."""
    gen = torch.Generator().manual_seed(13)
    counts = [(b * 7) % 4 if b % 5 else 0 for b in range(200)]
    counts[150] = 130
    starts, query, key, value = ragged(counts, 1, 2, 64, BF16, gen)
    got = prompt_attention(*(t.to(DEV) for t in (query, key, value)),
                           token_starts=starts.to(DEV), backend="hip")
    want, room = prompt64(query, key, value, starts, starts)
    assert_rows(got, want, room)
    # over longer keys, which are shared out
    lengths = [n + (b * 37) % 300 for b, n in enumerate(counts)]
    ends, _, key, value = ragged(lengths, 1, 1, 64, BF16, gen)
    got = prompt_attention(query.to(DEV), key.to(DEV), value.to(DEV), backend="hip",
                           token_starts=starts.to(DEV), key_starts=ends.to(DEV), window=200)
    want, room = prompt64(query, key, value, starts, ends, window=200)
    assert_rows(got, want, room)
