"""Rotary positions, the append to a paged cache and the decode over its
pages: the gfx950 kernels against the same in 64 bits (GPU).

The bounds are those of paged_math: 32-bit angles, products and sums, one
rounding to the inputs' type.
"""

import math

import pytest
import torch

from paged_math import assert_within, decode64, pages_for, rotate64
from refinekv import (PagedCache, Rotary, RotaryConfig, paged_append, paged_decode, rotate_heads)

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


def on_gpu(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def bits(t):
    return t.contiguous().view(torch.uint8)


# -- rotary ------------------------------------------------------------------

@pytest.mark.parametrize("tokens,heads,kv,dim,rotary_dim,interleaved,dtype", [
    (1, 32, 8, 128, 128, False, BF16), (8, 32, 8, 128, 128, False, BF16),
    (77, 28, 4, 128, 128, False, F16), (33, 5, 1, 96, 48, True, F16),
    (130, 4, 2, 64, 64, True, BF16), (19, 3, 3, 256, 64, False, F32),
    (7, 2, 1, 80, 40, False, BF16),   # half of the turning part no multiple of 8
    (9, 2, 1, 34, 6, True, F32), (5, 3, 2, 7, 6, False, BF16), (5, 3, 2, 7, 6, True, F16),
    (3, 2, 1, 700, 700, False, F32), (2, 1, 1, 2, 2, True, BF16), (300, 1, 1, 300, 2, False, F16),
    (21, 300, 9, 32, 32, False, BF16),  # more heads than a workgroup holds
    # parts of an odd number of vectors
    (40, 3, 1, 64, 40, True, BF16), (40, 3, 1, 72, 32, False, F16), (17, 6, 2, 88, 48, True, BF16),
    (25, 2, 1, 20, 12, True, F32), (25, 2, 2, 24, 16, False, F32),
    (2000, 17, 3, 128, 128, False, BF16),  # enough threads that each turns several heads
])
def test_rotate_heads(tokens, heads, kv, dim, rotary_dim, interleaved, dtype):
    gen = torch.Generator().manual_seed(tokens * 1000 + dim)
    query = torch.randn(tokens, heads, dim, generator=gen).to(dtype)
    key = torch.randn(tokens, kv, dim, generator=gen).to(dtype)
    positions = torch.randint(0, 131072, (tokens,), generator=gen)
    positions[0] = 131071
    config = RotaryConfig(head_dim=dim, rotary_dim=rotary_dim, base=500000.0,
                          interleaved=interleaved)
    q, k, p = on_gpu(query, key, positions)
    rotary = Rotary(config, DEV)
    for wide in (p, p.int()):
        got = rotate_heads(q, k, wide, rotary, backend="hip")
        for y, x, name in zip(got, (query, key), ("query", "key")):
            want, room = rotate64(x, positions, config.rates(), interleaved=interleaved)
            assert y.dtype == dtype and y.is_contiguous()
            assert_within(y, want, room, name)
    alone, none = rotate_heads(q, None, p, rotary, backend="hip")
    assert none is None and torch.equal(bits(alone), bits(got[0]))
    # the dims that pass are the inputs' own
    assert torch.equal(bits(got[0][..., rotary_dim:]), bits(q[..., rotary_dim:]))


@pytest.mark.parametrize("kwargs", [
    dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
    dict(scaling="llama3", factor=8.0, original_length=8192),
    dict(scaling="yarn", factor=4.0, original_length=32768),
    dict(scaling="yarn", factor=4.0, original_length=32768, attention_factor=0.7),
])
def test_rotate_heads_scalings_and_inverse(kwargs):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(40, 3, 128, generator=gen)
    positions = torch.randint(0, 1 << 20, (40,), generator=gen)
    config = RotaryConfig(head_dim=128, base=1000000.0, **kwargs)
    rotary = Rotary(config, DEV)
    scale = config.output_scale
    q, p = on_gpu(x, positions)
    for inverse in (False, True):
        got, _ = rotate_heads(q, None, p, rotary, inverse=inverse, backend="hip")
        want, room = rotate64(x, positions, config.rates(), scale, inverse=inverse)
        assert_within(got, want, room, str(inverse))
    # there and back: the factor twice, two roundings of fp32 data
    there, _ = rotate_heads(q, None, p, rotary, backend="hip")
    back, _ = rotate_heads(there, None, p, rotary, inverse=True, backend="hip")
    assert float((back.cpu() - x * scale ** 2).abs().max()) <= 40 * 2.0 ** -24 * scale ** 2 * float(
        x.abs().max())


def test_rotate_heads_negative_zero_and_far_positions():
    """Positions are any int64: 0 gives the input back bit for bit, negative
    ones turn back; a position of 2^31 - 1 keeps its angle to 2^-20 (its turns
    in fp64 have a step of 2^-24 at rate 1 / 2 pi)."""
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1))
    positions = torch.tensor([0, -5, 2 ** 31 - 1, -(2 ** 31) + 1])
    config = RotaryConfig(head_dim=64)
    got, _ = rotate_heads(x.to(DEV), None, positions.to(DEV), Rotary(config, DEV), backend="hip")
    want, room = rotate64(x, positions, config.rates())
    assert torch.equal(got[0].cpu(), x[0])
    assert_within(got[:2], want[:2], room[:2])
    assert float((got.cpu().double() - want)[2:].abs().max()) <= 2.0 ** -19 * float(x.abs().max())


def test_rotate_heads_views_and_in_place():
    """Rows inside a fused projection, heads and tokens in the other order,
    a reversed-stride-free unaligned view, and outputs over the inputs."""
    gen = torch.Generator().manual_seed(5)
    fused = torch.randn(50, 40, 64, generator=gen).to(BF16)
    positions = torch.arange(50)
    config = RotaryConfig(head_dim=64)
    rotary = Rotary(config, DEV)
    dev, pos = on_gpu(fused, positions)
    want = [rotate64(fused[:, a:b], positions, config.rates()) for a, b in ((0, 32), (32, 36))]
    got = rotate_heads(dev[:, :32], dev[:, 32:36], pos, rotary, backend="hip")
    for y, (w, room) in zip(got, want):
        assert_within(y, w, room)
    # (heads, tokens, dim) projections of a model, as its transposed view
    turned = dev[:, :32].transpose(0, 1).contiguous()
    y, _ = rotate_heads(turned.transpose(0, 1), None, pos, rotary, backend="hip")
    assert torch.equal(bits(y), bits(got[0]))
    # rows that start two bytes past any vector boundary
    odd = torch.empty(50 * 4 * 65 + 1, device=DEV, dtype=BF16)[1:].view(50, 4, 65)[..., :64]
    odd.copy_(dev[:, :4])
    y, _ = rotate_heads(odd, None, pos, rotary, backend="hip")
    assert torch.equal(bits(y), bits(got[0][:, :4]))
    # in place, the values beside them left alone
    rest = dev[:, 36:].clone()
    q, k = dev[:, :32], dev[:, 32:36]
    out = rotate_heads(q, k, pos, rotary, query_out=q, key_out=k, backend="hip")
    assert out[0].data_ptr() == dev.data_ptr()
    assert torch.equal(bits(dev[:, :32]), bits(got[0])) and torch.equal(bits(dev[:, 32:36]),
                                                                        bits(got[1]))
    assert torch.equal(bits(dev[:, 36:]), bits(rest))


def test_rotate_heads_no_tokens():
    q = torch.empty(0, 4, 64, device=DEV, dtype=BF16)
    out, key = rotate_heads(q, q[:, :2], torch.empty(0, device=DEV, dtype=torch.int64),
                            Rotary(RotaryConfig(head_dim=64), DEV), backend="hip")
    assert out.shape == (0, 4, 64) and key.shape == (0, 2, 64)


# -- append ------------------------------------------------------------------

def _append_case(lengths, new, page, heads, group, dim, dtype, seed, tail=0):
    """Inputs with ``tail`` rows behind the last sequence, the cache before,
    and each stored row's (token, page, row)."""
    gen = torch.Generator().manual_seed(seed)
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen)
    total = sum(new) + tail
    query, key, value = (torch.randn(total, n, dim, generator=gen).to(dtype)
                         for n in (heads * group, heads, heads))
    starts, places, positions, live = [0], [], [], []
    for b, (n, m) in enumerate(zip(lengths, new)):
        for j in range(m):
            p = n - m + j
            positions.append(max(p, 0))
            live.append(p >= 0)
            if p >= 0:
                places.append((starts[-1] + j, int(table[b, p // page]), p % page))
        starts.append(starts[-1] + m)
    positions += [0] * tail
    live += [False] * tail
    return dict(keys=keys, values=values, table=table, query=query, key=key, value=value,
                lengths=torch.tensor(lengths, dtype=torch.int32),
                starts=torch.tensor(starts, dtype=torch.int32), places=places,
                positions=torch.tensor(positions), live=torch.tensor(live))


def _check_append(case, config, cache, query, tail_of_query=True):
    """Every cell of the cache: new rows within rounding, the rest untouched."""
    keys, room = case["keys"].double(), torch.zeros(case["keys"].shape, dtype=torch.float64)
    values = case["values"].clone()
    if config is not None:
        scale = config.output_scale
        turned, slack = rotate64(case["key"], case["positions"], config.rates(), scale,
                                 config.interleaved)
    else:
        turned, slack = case["key"].double(), torch.zeros(case["key"].shape, dtype=torch.float64)
    for token, page, row in case["places"]:
        keys[page, :, row], room[page, :, row] = turned[token], slack[token]
        values[page, :, row] = case["value"][token]
    assert_within(cache.keys, keys, room, "keys")
    assert torch.equal(bits(cache.values.cpu()), bits(values))
    if query is not None:
        want, slack = rotate64(case["query"], case["positions"], config.rates(),
                               config.output_scale, config.interleaved)
        live = case["live"]
        assert_within(query[live.to(DEV)], want[live], slack[live], "query")
        assert torch.equal(bits(query.cpu()[~live]), bits(case["query"][~live]))


@pytest.mark.parametrize("lengths,page,heads,group,dim,rotary_dim,interleaved,dtype", [
    ([1], 16, 8, 4, 128, 128, False, BF16),
    ([1, 16, 17, 0, 300, 31, 32, 33], 16, 8, 4, 128, 128, False, BF16),
    ([129, 0, 64, 65, 1], 64, 4, 7, 128, 128, False, F16),
    ([5, 100], 32, 2, 1, 96, 24, True, F32), ([260, 256], 256, 1, 3, 10, 6, False, BF16),
    ([40] * 70, 16, 2, 2, 64, 32, True, BF16),
])
def test_append_one_token_each(lengths, page, heads, group, dim, rotary_dim, interleaved, dtype):
    """A decode step; a sequence of length 0 is an idle place."""
    case = _append_case(lengths, [1] * len(lengths), page, heads, group, dim, dtype, seed=dim)
    config = RotaryConfig(head_dim=dim, rotary_dim=rotary_dim, interleaved=interleaved,
                          base=500000.0)
    cache = PagedCache(*on_gpu(case["keys"], case["values"], case["table"], case["lengths"]))
    query = paged_append(*on_gpu(case["key"], case["value"]), cache, query=case["query"].to(DEV),
                         rotary=Rotary(config, DEV), backend="hip")
    _check_append(case, config, cache, query)


@pytest.mark.parametrize("lengths,new,tail,page,dtype", [
    ([100, 17, 64], [100, 1, 64], 0, 16, BF16), ([100, 0, 64, 0], [3, 0, 64, 0], 9, 32, F16),
    ([2, 50], [5, 50], 4, 16, F32),     # more new tokens than visible: the first have no place
    ([0, 0], [0, 0], 3, 16, BF16), ([700], [513], 0, 64, BF16),
])
def test_append_ragged_prompts(lengths, new, tail, page, dtype):
    case = _append_case(lengths, new, page, 2, 3, 64, dtype, seed=sum(lengths) + 1, tail=tail)
    config = RotaryConfig(head_dim=64, scaling="yarn", factor=4.0, original_length=64)
    cache = PagedCache(*on_gpu(case["keys"], case["values"], case["table"], case["lengths"]))
    query = case["query"].to(DEV)
    out = paged_append(*on_gpu(case["key"], case["value"]), cache, query=query, query_out=query,
                       rotary=Rotary(config, DEV), token_starts=case["starts"].to(DEV),
                       backend="hip")
    assert out is query
    _check_append(case, config, cache, out)


def test_append_without_rotation_and_other_cache_layouts():
    """Keys as they are; a cache kept as (pages, page_size, heads, dim), and
    one whose keys and values lie in one tensor."""
    case = _append_case([33, 5, 70], [33, 2, 1], 16, 3, 2, 64, BF16, seed=8)
    table, lengths, starts = on_gpu(case["table"], case["lengths"], case["starts"])
    key, value = on_gpu(case["key"], case["value"])
    for layout in ("rows", "both"):
        if layout == "rows":
            keys, values = (case[n].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
                            for n in ("keys", "values"))
        else:
            both = torch.stack([case["keys"], case["values"]], 1).to(DEV)
            keys, values = both[:, 0], both[:, 1]
        cache = PagedCache(keys, values, table, lengths)
        assert paged_append(key, value, cache, token_starts=starts, backend="hip") is None
        _check_append(case, None, cache, None)


def test_append_bad_pages_and_short_tables_store_nothing():
    """A page outside the cache or a position past the table: that row is
    dropped, the others and the queries are as ever."""
    case = _append_case([20, 20, 20], [20, 20, 20], 16, 2, 1, 32, BF16, seed=4)
    table = case["table"].clone()
    table[0, 1], table[1, 0] = -7, case["keys"].shape[0]
    case["places"] = [(t, p, r) for t, p, r in case["places"]
                      if not (16 <= t < 20 or 20 <= t < 36)]
    lengths = case["lengths"].clone()
    config = RotaryConfig(head_dim=32)
    cache = PagedCache(*on_gpu(case["keys"], case["values"], table, lengths))
    query = paged_append(*on_gpu(case["key"], case["value"]), cache, query=case["query"].to(DEV),
                         rotary=Rotary(config, DEV), token_starts=case["starts"].to(DEV),
                         backend="hip")
    _check_append(case, config, cache, query)
    # a table of one block: tokens 16.. of each sequence have no page
    case = _append_case([20, 20], [20, 20], 16, 2, 1, 32, BF16, seed=6)
    case["places"] = [(t, p, r) for t, p, r in case["places"] if t % 20 < 16]
    cache = PagedCache(*on_gpu(case["keys"], case["values"], case["table"][:, :1].contiguous(),
                               case["lengths"]))
    paged_append(*on_gpu(case["key"], case["value"]), cache, rotary=Rotary(config, DEV),
                 token_starts=case["starts"].to(DEV), backend="hip")
    _check_append(case, config, cache, None)


# -- decode ------------------------------------------------------------------

def _decode(case, group, scaling=None, workspace=None, **kwargs):
    query, keys, values, table, lengths = on_gpu(*case)
    cache = PagedCache(keys, values, table, lengths)
    return paged_decode(query, cache, scaling=scaling, workspace=workspace, backend="hip",
                        **kwargs)


def _decode_case(lengths, page, heads, group, dim, dtype, seed, peak=0.0, **over):
    gen = torch.Generator().manual_seed(seed)
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen, **over)
    query = torch.randn(len(lengths), heads * group, dim, generator=gen).to(dtype)
    if peak:
        # some tokens along the queries: a softmax with few large weights
        for b, n in enumerate(lengths):
            for t in range(b % 5, n, 17):
                toward = query[b].view(heads, group, dim)[:, t % group].float() * peak
                at = int(table[b, t // page]), slice(None), t % page
                keys[at] = (keys[at].float() + toward).to(dtype)
    return query, keys, values, table, torch.tensor(lengths, dtype=torch.int32)


@pytest.mark.parametrize("lengths,page,heads,group,dim,dtype", [
    ([1], 16, 1, 1, 32, BF16), ([1, 2, 15, 16, 17], 16, 2, 4, 64, F16),
    ([2003], 16, 8, 4, 128, BF16), ([31, 32, 33, 63, 64, 65, 0, 127, 128, 129], 32, 2, 4, 128, BF16),
    ([0, 0, 0], 16, 2, 2, 64, BF16), ([700, 0, 1, 1300], 64, 4, 7, 128, F16),
    ([255, 256, 257], 256, 1, 16, 256, BF16), ([900, 100], 128, 3, 5, 160, F16),
    ([333, 1], 16, 2, 2, 96, BF16), ([500], 32, 1, 9, 192, F16), ([77, 400], 16, 1, 3, 224, BF16),
    ([50 + 13 * b for b in range(40)], 16, 2, 8, 64, BF16), ([4000], 16, 1, 1, 128, BF16),
    ([3, 0] * 90, 16, 3, 2, 32, BF16), ([3, 0, 40] * 200, 16, 1, 2, 32, F16),
    ([20000, 7], 16, 2, 3, 64, BF16), ([9000, 9000], 64, 3, 1, 256, BF16),
])
def test_decode(lengths, page, heads, group, dim, dtype):
    case = _decode_case(lengths, page, heads, group, dim, dtype, seed=sum(lengths) + dim,
                        peak=0.5)
    got = _decode(case, group)
    want, room = decode64(*case, dim ** -0.5)
    assert got.dtype == dtype and got.shape == case[0].shape
    assert_within(got, want, room)


def test_decode_scaling_strided_query_and_cache_layouts():
    heads, group, dim, lengths = 2, 3, 64, [40, 129, 7]
    case = _decode_case(lengths, 32, heads, group, dim, BF16, seed=2)
    want, room = decode64(*case, 0.3)
    got = _decode(case, group, scaling=0.3)
    assert_within(got, want, room)
    query, keys, values, table, lens = on_gpu(*case)
    other = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (keys, values)]
    assert torch.equal(bits(paged_decode(query, PagedCache(*other, table, lens), scaling=0.3,
                                         backend="hip")), bits(got))
    both = torch.stack([values, keys], 2).transpose(0, 1)  # (heads, pages, 2, page, dim) views
    views = [both[:, :, i].transpose(0, 1) for i in (1, 0)]
    wide = torch.zeros(3, heads * group + 5, dim, device=DEV, dtype=BF16)
    wide[:, 2:2 + heads * group] = query
    out = torch.empty_like(query)
    result = paged_decode(wide[:, 2:2 + heads * group], PagedCache(*views, table, lens),
                          scaling=0.3, output=out, backend="hip")
    assert result is out and torch.equal(bits(out), bits(got))


def test_decode_masked_infinities_and_nan_inputs():
    """What no sequence sees is never read into a result (pages_for fills it
    with NaN; here with infinities too); what is seen counts: a NaN key or
    value, a score of -inf everywhere (0 / 0) or of +inf, as a softmax has it."""
    heads, group, dim = 1, 2, 32
    query, keys, values, table, lengths = _decode_case([20, 40, 40, 40, 40, 30], 16, heads, group,
                                                       dim, BF16, seed=9)
    hidden = keys.isnan()
    keys[hidden] = math.inf
    values[hidden] = -math.inf
    case = (query, keys, values, table, lengths)
    want, room = decode64(*case, 0.2)
    assert_within(_decode(case, group, scaling=0.2), want, room)
    keys[int(table[1, 1]), 0, 3, 5] = math.nan          # every row of sequence 1
    values[int(table[2, 2]), 0, 1, 7] = math.nan        # dim 7 of sequence 2
    query[3, :, 0] = 1.0
    query[4, :, 0] = 1.0
    for j in range(3):
        keys[int(table[3, j]), 0, :, 0] = -math.inf     # every score of sequence 3
    keys[int(table[4, 0]), 0, 2, 0] = -math.inf         # one score of sequence 4
    got = _decode(case, group, scaling=0.2).cpu()
    want, room = decode64(*case, 0.2)
    assert want[1].isnan().all() and want[3].isnan().all()
    assert want[2, :, 7].isnan().all() and not want[2, :, :7].isnan().any()
    room[4] = torch.where(room[4].isnan() | room[4].isinf(), 0.0, room[4])
    clean = torch.ones(6, dtype=torch.bool)
    clean[4] = False
    assert_within(got[clean], want[clean], room[clean])
    # sequence 4 as if the token were not there
    take = table[4, :3].long()
    k, v = (t[take, 0].reshape(-1, dim)[:40].double() for t in (keys, values))
    keep = torch.arange(40) != 2
    k, v = k[keep], v[keep]
    p = torch.softmax(query[4].double() @ k.T * 0.2, -1)
    assert_within(got[4], p @ v, 2.0 ** -8 * (p @ v).abs() + 2.0 ** -14 * (p @ v.abs()))


def test_decode_bad_pages_and_lengths_give_nan_rows_of_their_sequence():
    heads, group, dim = 2, 2, 64
    query, keys, values, table, lengths = _decode_case([50, 50, 50, 50, 300], 16, heads, group,
                                                       dim, BF16, seed=12)
    table[0, 3], table[1, 0] = -1, keys.shape[0]
    lengths[2] = table.shape[1] * 16 + 1
    case = (query, keys, values, table, lengths)
    want, room = decode64(*case, dim ** -0.5)
    assert want[:3].isnan().all() and not want[3:].isnan().any()
    assert_within(_decode(case, group), want, room)


def test_decode_repeats_bit_for_bit_and_workspaces_are_reusable():
    """One workspace through calls of different shapes, and the same call
    again: the same bits each time."""
    workspace, first = {}, {}
    shapes = [([2003], 16, 8, 4, 128, BF16), ([30, 0, 4000, 700], 32, 4, 7, 128, F16),
              ([5] * 30, 16, 2, 2, 64, BF16), ([9000, 20], 64, 1, 16, 256, BF16)]
    for again in range(3):
        for i, (lengths, page, heads, group, dim, dtype) in enumerate(shapes):
            case = _decode_case(lengths, page, heads, group, dim, dtype, seed=40 + i)
            got = _decode(case, group, workspace=workspace)
            assert torch.equal(bits(got), bits(first.setdefault(i, got.clone()))), (again, i)


def test_decode_fp16_keeps_many_small_weights():
    """One key that outweighs each of 60000 others by 2^24 or more: together
    the others still weigh, though each is below fp16's subnormals against 1."""
    length, dim = 60001, 32
    query = torch.zeros(1, 1, dim, dtype=F16)
    query[0, 0, 0] = 1.0
    blocks = -(-length // 256)
    keys = torch.zeros(blocks, 1, 256, dim, dtype=F16)
    values = torch.full((blocks, 1, 256, dim), -1.0, dtype=F16)
    values[7, 0, 100] = 1.0
    lengths = torch.tensor([length], dtype=torch.int32)
    table = torch.arange(blocks, dtype=torch.int32)[None]
    for above in (17.0, 19.0, 23.0):
        keys[7, 0, 100, 0] = above
        case = (query, keys, values, table, lengths)
        want, room = decode64(*case, 1.0)
        others = 60000 * math.exp(-above)
        assert abs(float(want[0, 0, 0]) - (1 - others) / (1 + others)) < 1e-9
        assert_within(_decode(case, 1, scaling=1.0), want, room, str(above))


def test_decode_nan_query_stays_in_its_row():
    case = _decode_case([300, 40], 16, 2, 4, 64, BF16, seed=14)
    clean = _decode(case, 4).cpu()
    case[0][0, 5, 3] = math.nan
    got = _decode(case, 4).cpu()
    assert got[0, 5].isnan().all()
    got[0, 5] = clean[0, 5]
    assert torch.equal(bits(got), bits(clean))


def test_decode_many_sequences():
    """More sequences than a wave has lanes, many of them idle."""
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(-2, 60, (3000,), generator=gen).clamp_min(0).tolist()
    case = _decode_case(lengths, 16, 1, 1, 32, BF16, seed=15)
    want, room = decode64(*case, 32 ** -0.5)
    assert_within(_decode(case, 1), want, room)


def test_offsets_past_32_bits():
    """A cache of 2^32 elements and more a tensor: the first and last pages,
    written and read."""
    heads, page, dim = 8, 16, 128
    pages = (1 << 32) // (heads * page * dim) + 5
    keys, values = (torch.empty(pages, heads, page, dim, device=DEV, dtype=BF16) for _ in range(2))
    places = [pages - 1, 0, pages - 3, 131073, pages - 2]
    table = torch.tensor([places], dtype=torch.int32, device=DEV)
    length = 5 * page - 3
    cache = PagedCache(keys, values, table,
                       torch.tensor([length], dtype=torch.int32, device=DEV))
    gen = torch.Generator().manual_seed(21)
    key, value = (torch.randn(length, heads, dim, generator=gen).to(BF16) for _ in range(2))
    query = torch.randn(1, heads * 4, dim, generator=gen).to(BF16)
    starts = torch.tensor([0, length], dtype=torch.int32, device=DEV)
    paged_append(*on_gpu(key, value), cache, token_starts=starts, backend="hip")
    got = paged_decode(query.to(DEV), cache, backend="hip")
    small = [t[places].cpu() for t in (keys, values)]
    for t, rows in zip(small, (key, value)):
        held = t.transpose(1, 2).reshape(-1, heads, dim)[:length]
        assert torch.equal(bits(held), bits(rows))
    want, room = decode64(query, *small, torch.arange(5, dtype=torch.int32)[None], [length],
                          dim ** -0.5)
    assert_within(got, want, room)


# -- together ----------------------------------------------------------------

def _serving_batch(seed, page=16, heads=2, group=4, dim=64, dtype=BF16):
    """A cache filled by ragged prompts, and room for more tokens."""
    gen = torch.Generator().manual_seed(seed)
    prompts = [37, 5, 0, 120]
    cache = PagedCache.empty(40, heads, page, dim, len(prompts), 12, dtype=dtype, device=DEV)
    cache.block_table.copy_(torch.randperm(40, generator=gen)[:40].int().view(4, 10).to(DEV)
                            .repeat(1, 2)[:, :12])
    cache.block_table[:, 10:] = -1
    config = RotaryConfig(head_dim=dim, base=500000.0)
    rows = lambda n, h: torch.randn(n, h, dim, generator=gen).to(dtype)  # noqa: E731
    return cache, config, prompts, rows


def test_prompts_then_decode_steps_match_a_contiguous_softmax():
    """Prompts appended, then steps of append and decode.  Each step's outputs
    are the attention over the cache as it then stands, and at the end the
    cache holds every key turned to its position, in order, and every value."""
    cache, config, prompts, rows = _serving_batch(1)
    heads, group, dim = cache.heads, 4, cache.head_dim
    rotary, workspace = Rotary(config, DEV), {}
    total = sum(prompts)
    key, value = rows(total, heads), rows(total, heads)
    starts = torch.tensor([0, *torch.tensor(prompts).cumsum(0).tolist()], dtype=torch.int32)
    cache.lengths.copy_(torch.tensor(prompts, dtype=torch.int32))
    assert paged_append(*on_gpu(key, value), cache, rotary=rotary, token_starts=starts.to(DEV),
                        backend="hip") is None
    history = [[key[starts[b]:starts[b + 1]], value[starts[b]:starts[b + 1]]] for b in range(4)]
    active = torch.tensor([1, 1, 0, 1], dtype=torch.int32, device=DEV)  # sequence 2 is idle
    for _ in range(20):
        key, value, query = rows(4, heads), rows(4, heads), rows(4, heads * group)
        cache.lengths.add_(active)
        turned = paged_append(*on_gpu(key, value), cache, query=query.to(DEV), rotary=rotary,
                              backend="hip")
        out = paged_decode(turned, cache, workspace=workspace, backend="hip").cpu()
        assert (out[2] == 0).all()
        for b in (0, 1, 3):
            history[b] = [torch.cat([h, x[b:b + 1]]) for h, x in zip(history[b], (key, value))]
        want, room = decode64(turned.cpu(), cache.keys.cpu(), cache.values.cpu(),
                              cache.block_table.cpu(), cache.lengths.cpu(), dim ** -0.5)
        assert_within(out, want, room)
    for b in (0, 1, 3):
        n = len(history[b][0])
        assert n == int(cache.lengths[b])
        take = cache.block_table[b, :-(-n // 16)].long()
        held, same = (t[take].transpose(1, 2).reshape(-1, heads, dim)[:n].cpu()
                      for t in (cache.keys, cache.values))
        want, room = rotate64(history[b][0], torch.arange(n), config.rates())
        assert_within(held, want, room)
        assert torch.equal(bits(same), bits(history[b][1]))


def test_graph_replays_of_append_and_decode_match_eager_steps():
    """One captured step (lengths, append, decode), replayed with other
    inputs and eager work in between, against the same steps called eagerly."""
    results = []
    for graphed in (False, True):
        cache, config, prompts, rows = _serving_batch(2)
        heads, group = cache.heads, 4
        rotary, workspace = Rotary(config, DEV), {}
        cache.lengths.copy_(torch.tensor(prompts, dtype=torch.int32))
        cache.keys.normal_(generator=torch.Generator(DEV).manual_seed(3))
        cache.values.normal_(generator=torch.Generator(DEV).manual_seed(4))
        key, value = (torch.zeros(4, heads, 64, device=DEV, dtype=BF16) for _ in range(2))
        query = torch.zeros(4, heads * group, 64, device=DEV, dtype=BF16)
        out, turned = torch.empty_like(query), torch.empty_like(query)

        def step():
            cache.lengths.add_(1)
            paged_append(key, value, cache, query=query, rotary=rotary, query_out=turned,
                         backend="hip")
            paged_decode(turned, cache, workspace=workspace, output=out, backend="hip")

        step()  # sizes the workspace
        cache.lengths.sub_(1)
        torch.cuda.synchronize()
        if graphed:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        outs = []
        for _ in range(6):
            key.copy_(rows(4, heads))
            value.copy_(rows(4, heads))
            query.copy_(rows(4, heads * group))
            graph.replay() if graphed else step()
            outs.append(out.clone())
            torch.cuda.synchronize()
        results.append((outs, cache.keys.clone(), cache.values.clone(), cache.lengths.clone()))
    for a, b in zip(results[0][0], results[1][0]):
        assert torch.equal(bits(a), bits(b))
    for a, b in zip(results[0][1:], results[1][1:]):
        assert torch.equal(bits(a), bits(b))


def test_graphs_of_two_shapes_share_a_workspace():
    """Two captured calls whose scratch differs in size keep theirs: replays
    in turn, with eager work between, give the eager results."""
    workspace, runs = {}, []
    for seed, (lengths, heads, group, dim) in enumerate((([900, 30], 2, 4, 64),
                                                         ([70, 0, 2000], 1, 16, 128))):
        case = _decode_case(lengths, 16, heads, group, dim, BF16, seed=60 + seed)
        query, *parts = on_gpu(*case)
        cache, out = PagedCache(*parts), torch.empty_like(query)
        want = paged_decode(query, cache, workspace=workspace, backend="hip")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_decode(query, cache, workspace=workspace, output=out, backend="hip")
        runs.append((graph, out, want, query, cache))
    for _ in range(4):
        for graph, out, want, query, cache in runs:
            out.zero_()
            junk = torch.randn(1 << 20, device=DEV)  # takes memory that was let go
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(want)) and bool(junk.isfinite().all())


def test_append_no_tokens():
    cache = PagedCache.empty(4, 2, 16, 64, 3, 2, device=DEV)
    rows = torch.empty(0, 2, 64, device=DEV, dtype=BF16)
    starts = torch.zeros(4, device=DEV, dtype=torch.int32)
    out = paged_append(rows, rows, cache, query=rows, rotary=Rotary(RotaryConfig(head_dim=64), DEV),
                       token_starts=starts, backend="hip")
    assert out.shape == (0, 2, 64) and not cache.keys.any()


def test_unsupported_shapes_take_torch_or_are_refused():
    """auto answers what the kernels do not take; an explicit request says why."""
    for heads, group, dim, dtype in ((1, 17, 64, BF16), (2, 2, 48, BF16), (2, 2, 64, F32)):
        query, *parts = on_gpu(*_decode_case([40, 0, 17], 16, heads, group, dim, dtype, seed=dim))
        cache = PagedCache(*parts)
        with pytest.raises(TypeError):
            paged_decode(query, cache, backend="hip")
        got = paged_decode(query, cache)
        want, room = decode64(query.cpu(), *(t.cpu() for t in parts), dim ** -0.5)
        assert_within(got, want, room + 2.0 ** -12 * want.abs())
    x = torch.randn(5, 2, 64, device=DEV, dtype=torch.float64)
    positions = torch.arange(5, device=DEV)
    config = RotaryConfig(head_dim=64)
    with pytest.raises(TypeError):
        rotate_heads(x, None, positions, Rotary(config, DEV), backend="hip")
    got, _ = rotate_heads(x, None, positions, Rotary(config, DEV))
    want, _ = rotate64(x.cpu(), positions.cpu(), config.rates())
    assert float((got.cpu() - want).abs().max()) < 1e-12


def test_two_streams_at_once():
    """Calls of two streams with a workspace each, interleaved."""
    runs = []
    for seed, shape in enumerate((([3000, 10], 16, 8, 4, 128, BF16), ([700] * 9, 32, 2, 7, 64, F16))):
        lengths, page, heads, group, dim, dtype = shape
        query, *parts = on_gpu(*_decode_case(lengths, page, heads, group, dim, dtype, seed=70 + seed))
        cache = PagedCache(*parts)
        runs.append((query, cache, paged_decode(query, cache, backend="hip"), {},
                     torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(8):
        for query, cache, _, workspace, stream, outs in runs:
            with torch.cuda.stream(stream):
                outs.append(paged_decode(query, cache, workspace=workspace, backend="hip"))
    torch.cuda.synchronize()
    for _, _, want, _, _, outs in runs:
        assert all(torch.equal(bits(out), bits(want)) for out in outs)


def test_unaligned_cache():
    """A cache that starts two bytes past any vector boundary: the append
    writes it element by element, the decode leaves it to torch or says why."""
    case = _append_case([20, 5], [20, 5], 16, 2, 2, 64, BF16, seed=50)
    shape = case["keys"].shape
    keys, values = (torch.empty(case["keys"].numel() + 1, device=DEV, dtype=BF16)[1:].view(shape)
                    .copy_(case[n]) for n in ("keys", "values"))
    table, lengths, starts = on_gpu(case["table"], case["lengths"], case["starts"])
    cache = PagedCache(keys, values, table, lengths)
    config = RotaryConfig(head_dim=64)
    query = paged_append(*on_gpu(case["key"], case["value"]), cache, query=case["query"].to(DEV),
                         rotary=Rotary(config, DEV), token_starts=starts, backend="hip")
    _check_append(case, config, cache, query)
    last = torch.stack([query[19], query[24]])
    with pytest.raises(TypeError):
        paged_decode(last, cache, backend="hip")
    got = paged_decode(last, cache)
    want, room = decode64(last.cpu(), keys.cpu(), values.cpu(), case["table"], case["lengths"],
                          64 ** -0.5)
    assert_within(got, want, room + 2.0 ** -12 * want.abs())
    # an unaligned query is copied
    aligned = [t.clone() for t in (keys, values)]
    odd = torch.empty(last.numel() + 1, device=DEV, dtype=BF16)[1:].view(last.shape).copy_(last)
    cache = PagedCache(*aligned, table, lengths)
    assert torch.equal(bits(paged_decode(odd, cache, backend="hip")),
                       bits(paged_decode(last, cache, backend="hip")))


def test_strides_of_single_places_are_not_read():
    """Views keep any stride on an axis of length one; with odd ones there the
    calls answer as without."""
    case = _decode_case([13], 16, 1, 1, 64, BF16, seed=52, spare=0)
    query, keys, values, table, lengths = on_gpu(*case)
    assert keys.shape == (1, 1, 16, 64)
    want = paged_decode(query, PagedCache(keys, values, table, lengths), backend="hip")
    odd = lambda t: t.as_strided(t.shape, (3, 5, 64, 1))  # noqa: E731
    cache = PagedCache(odd(keys), odd(values), table, lengths)
    got = paged_decode(query.as_strided((1, 1, 64), (7, 9, 1)), cache, backend="hip")
    assert torch.equal(bits(got), bits(want))
    rotary = Rotary(RotaryConfig(head_dim=64), DEV)
    row = torch.randn(1, 1, 64, device=DEV).to(BF16)
    turned = paged_append(row.as_strided((1, 1, 64), (3, 1, 1)), row, cache, query=row,
                          rotary=rotary, backend="hip")
    position = torch.tensor([12], device=DEV)
    alone, _ = rotate_heads(row.as_strided((1, 1, 64), (1, 3, 1)), None, position, rotary,
                            backend="hip")
    place = keys[int(table[0, 0]), 0, 12]
    assert torch.equal(bits(turned), bits(alone)) and torch.equal(bits(place), bits(alone[0, 0]))


def test_copies_of_a_cache_are_their_own():
    import copy

    case = _decode_case([40, 3], 16, 2, 2, 64, BF16, seed=51)
    query, *parts = on_gpu(*case)
    cache = PagedCache(*parts)
    want = paged_decode(query, cache, backend="hip")
    other = copy.deepcopy(cache)
    cache.keys.zero_()
    assert torch.equal(bits(paged_decode(query, other, backend="hip")), bits(want))
    assert not torch.equal(bits(paged_decode(query, copy.copy(cache), backend="hip")), bits(want))


def test_calls_on_another_stream():
    case = _decode_case([500, 30], 16, 2, 4, 64, BF16, seed=31)
    want = _decode(case, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _decode(case, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(bits(got), bits(want))


def test_rotate_and_append_agree_bit_for_bit():
    """The same kernel behind both entries."""
    case = _append_case([64], [64], 16, 2, 2, 128, F16, seed=77)
    config = RotaryConfig(head_dim=128)
    rotary = Rotary(config, DEV)
    cache = PagedCache(*on_gpu(case["keys"], case["values"], case["table"], case["lengths"]))
    query, key, value, starts = on_gpu(case["query"], case["key"], case["value"], case["starts"])
    turned = paged_append(key, value, cache, query=query, rotary=rotary, token_starts=starts,
                          backend="hip")
    q, k = rotate_heads(query, key, torch.arange(64, device=DEV), rotary, backend="hip")
    assert torch.equal(bits(turned), bits(q))
    stored = cache.keys[cache.block_table[0, :4].long()].transpose(1, 2).reshape(64, 2, 128)
    assert torch.equal(bits(stored), bits(k))
