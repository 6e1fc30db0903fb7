"""The paged cache in 4 bits on the CPU: the format, the order of its bytes, the
torch restatement against the same in 64 bits, and the refusals; the options of
the decode's scores."""

import copy
import math

import pytest
import torch

from paged_math import assert_within, pages_for
from quantized_math import attend64, decode64_quantized, quantize64
from refinekv import (PagedCache, QuantizedCache, Rotary, RotaryConfig, paged_append, paged_decode,
                      paged_read, quantized, rotate_heads)

BF16, F16 = torch.bfloat16, torch.float16


def held(rows):
    codes, scale, zero = quantize64(rows)
    return torch.from_numpy(zero + scale * codes)


def same(got, want):
    """Equal values, NaN in the same places."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.5),
                                                                  want.nan_to_num(0.5))


# -- the format --------------------------------------------------------------

@pytest.mark.parametrize("dim", range(32, 257, 32))
def test_order_of_codes_and_scales(dim):
    """Every code where the kernels look for it, and back."""
    gen = torch.Generator().manual_seed(dim)
    codes = torch.randint(0, 16, (2, 3, 16, dim), generator=gen, dtype=torch.uint8)
    scales = torch.randn(2, 3, 16, dim // 32, 2, generator=gen).half()
    keys, values = quantized.pack_keys(codes), quantized.pack_values(codes)
    assert torch.equal(quantized.unpack_keys(keys), codes)
    assert torch.equal(quantized.unpack_values(values), codes)
    assert torch.equal(quantized.unpack_scales(quantized.pack_scales(scales)), scales)
    groups, row = dim // 32, keys[1, 2, 7].numpy().view("<u4")
    block = values[0, 1].reshape(4, 2 * dim)[2].numpy()
    pairs = quantized.pack_scales(scales)[1, 0].reshape(4, groups, 8)
    for d in range(dim):
        lane, entry = d % 32 // 8, d % 8
        shift = 4 * (entry // 2) + 16 * (entry % 2)
        assert int(row[lane * groups + d // 32]) >> shift & 15 == int(codes[1, 2, 7, d])
        first, each = next((f, e) for f, e in quantized._pieces(dim)[::-1] if d >= f)
        words = block[2 * first:2 * first + 32 * each].view("<u4")
        column, inside = divmod(d - first, each)
        for token in range(4):
            m = token // 2 * each + inside
            shift = 4 * (m % 4) + 16 * (token % 2)
            assert int(words[column * each // 2 + m // 4]) >> shift & 15 == int(
                codes[0, 1, 8 + token, d])
            assert pairs[3, d // 32, token] == scales[1, 0, 12 + token, d // 32, 0]
            assert pairs[3, d // 32, 4 + token] == scales[1, 0, 12 + token, d // 32, 1]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [1.0, 300.0, 2.0 ** -9])
def test_quantize_is_the_definition(dtype, size):
    x = (torch.randn(500, 3, 64, generator=torch.Generator().manual_seed(1)) * size).to(dtype)
    x[0] = x[0].abs() + 50 * size  # far from 0
    x[1] = 3.5  # a group of one value: scale 0
    x[2, 0, 3], x[2, 1, 40], x[2, 2, 5] = math.nan, math.inf, 4128.0  # not held
    x[3, 0, :2] = torch.tensor([4096.0, -4096.0])
    codes, scales = quantized.quantize(x)
    want, scale, zero = (torch.from_numpy(t) for t in quantize64(x))
    assert torch.equal(codes.double(), want)
    assert same(scales[..., 0].double(), scale[..., ::32])
    assert same(scales[..., 1].double(), zero[..., ::32])
    value = quantized.dequantize(codes, scales).double()
    assert same(value, zero + scale * want)
    off = (value - x.double()).abs()
    live = ~value.isnan()
    groups = x.double().unflatten(-1, (-1, 32))
    assert torch.equal(live, (groups.isfinite() & (groups.abs() <= 4096)).all(-1, keepdim=True)
                       .expand_as(groups).flatten(-2))
    assert not bool(live[2].all()) and bool(live[3:].any())
    # half a scale, and the roundings of zero and scale to fp16 (scales round up after it)
    room = scale / 2 + x.double().abs() * 2.0 ** -11 + 15 * scale * 2.0 ** -11 + 2.0 ** -19
    assert bool((off <= room)[live].all())
    assert bool((value[1] == 3.5).all())
    bits = scales[..., 0].contiguous().view(torch.int16)
    assert bool((bits[~scales[..., 0].isnan()] & 15 == 0).all())


def test_packed_and_unpacked():
    gen = torch.Generator().manual_seed(2)
    codes = [torch.randint(0, 16, (3, 2, 16, 96), generator=gen, dtype=torch.uint8)
             for _ in range(2)]
    scales = [torch.randn(3, 2, 16, 3, 2, generator=gen).half() for _ in range(2)]
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cache = QuantizedCache.packed(*codes, *scales, table, lengths, dtype=F16)
    assert (cache.head_dim, cache.page_size, cache.heads, cache.pages) == (96, 16, 2, 3)
    assert cache.dtype == F16 and cache.capacity == 32
    for got, want in zip(cache.unpacked(), (*codes, *scales)):
        assert torch.equal(got, want)
    again = copy.deepcopy(cache)
    assert again.key_codes.data_ptr() != cache.key_codes.data_ptr()


# -- append and read ---------------------------------------------------------

def _rows(tokens, heads, dim, dtype, gen):
    return torch.randn(tokens, heads, dim, generator=gen).to(dtype)


@pytest.mark.parametrize("dim,dtype,page", [(128, BF16, 16), (96, F16, 32), (32, BF16, 16)])
def test_append_and_read_torch(dim, dtype, page):
    gen = torch.Generator().manual_seed(dim)
    cache = QuantizedCache.empty(9, 2, page, dim, 4, 3, dtype=dtype)
    for t in (cache.key_codes, cache.value_codes):  # as earlier calls left them
        t.copy_(torch.randint(0, 256, t.shape, generator=gen, dtype=torch.uint8))
    cache.block_table.copy_(torch.tensor([[5, 1, -1], [2, 7, 4], [-1, -1, -1], [3, 9, 0]]))
    lengths = [page + 3, 2 * page + 1, 0, page + 2]  # sequence 3: its second page is not there
    new = [page + 3, 5, 0, 4]
    cache.lengths.copy_(torch.tensor(lengths))
    starts = torch.tensor([0] + new).cumsum(0).int()
    tokens = int(starts[-1]) + 2  # two rows of no sequence
    key, value = (_rows(tokens, 2, dim, dtype, gen) for _ in range(2))
    query = _rows(tokens, 6, dim, dtype, gen)
    rotary = Rotary(RotaryConfig(head_dim=dim))
    before = [t.clone() for t in cache.unpacked()]
    turned = paged_append(key, value, cache, query=query, rotary=rotary, token_starts=starts)
    position, want, stored = [], [before[0].clone(), before[1].clone()], []
    for b, n in enumerate(new):
        position += range(lengths[b] - n, lengths[b])
    position += [0, 0]
    q, k = rotate_heads(query, key, torch.tensor(position), rotary)
    assert torch.equal(turned[:-2], q[:-2]) and torch.equal(turned[-2:], query[-2:])
    codes = [torch.from_numpy(quantize64(t)[0]).to(torch.uint8) for t in (k, value)]
    for b, n in enumerate(new):
        for i in range(n):
            row, at = int(starts[b]) + i, lengths[b] - n + i
            page_of = int(cache.block_table[b, at // page])
            if 0 <= page_of < cache.pages:
                stored.append(row)
                for pool, c in zip(want, codes):
                    pool[page_of, :, at % page] = c[row]
    got = cache.unpacked()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    keys, values = paged_read(cache, tokens, token_starts=starts)
    assert keys.dtype == dtype and keys.shape == key.shape
    for out, rows in ((keys, k), (values, value)):
        assert torch.equal(out[stored].double(), held(rows)[stored].to(dtype).double())
        lost = [r for r in range(tokens - 2) if r not in stored]
        assert lost and bool(out[lost].isnan().all()) and not bool(out[-2:].any())


def test_read_of_a_16_bit_cache_torch():
    gen = torch.Generator().manual_seed(4)
    cache = PagedCache.empty(4, 3, 16, 40, 2, 2, dtype=torch.float32)
    cache.block_table.copy_(torch.tensor([[2, 0], [3, -1]]))
    cache.lengths.copy_(torch.tensor([20, 18]))
    starts = torch.tensor([0, 20, 38], dtype=torch.int32)
    key, value = (torch.randn(39, 3, 40, generator=gen) for _ in range(2))
    paged_append(key, value, cache, token_starts=starts)
    keys, values = paged_read(cache, 39, token_starts=starts)
    for out, rows in ((keys, key), (values, value)):
        assert torch.equal(out[:36], rows[:36])
        assert bool(out[36:38].isnan().all()) and not bool(out[38:].any())
    last = paged_read(cache, 2)[0]
    assert torch.equal(last[0], key[19]) and bool(last[1].isnan().all())


# -- decode ------------------------------------------------------------------

def quantized_pages(lengths, page, heads, dim, dtype, gen, **kwargs):
    """(cache, (codes, scales, zeros) pairs in 64 bits): pages of randn, NaN in
    every row no sequence sees."""
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen, **kwargs)
    plain = [quantized.quantize(t) for t in (keys, values)]
    cache = QuantizedCache.packed(plain[0][0], plain[1][0], plain[0][1], plain[1][1], table,
                                  torch.tensor(lengths, dtype=torch.int32), dtype=dtype)
    wide = [quantize64(t) for t in (keys, values)]
    return cache, [tuple(torch.from_numpy(w[i]) for w in wide) for i in range(3)]


@pytest.mark.parametrize("options", [
    {}, dict(softcap=5.0), dict(window=7), dict(window=40, softcap=30.0), dict(slopes=True)])
@pytest.mark.parametrize("dim,dtype,group", [(64, BF16, 3), (96, F16, 1)])
def test_decode_torch(dim, dtype, group, options):
    gen = torch.Generator().manual_seed(dim)
    lengths = [1, 0, 37, 64, -3]
    cache, wide = quantized_pages(lengths, 16, 2, dim, dtype, gen)
    query = _rows(5, 2 * group, dim, dtype, gen)
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.linspace(0.5, 0.01, 2 * group)
    got = paged_decode(query, cache, **options)
    want, room = decode64_quantized(query, *wide, cache.block_table, lengths, dim ** -0.5,
                                    **options)
    assert_within(got, want, room)


@pytest.mark.parametrize("options", [dict(softcap=20.0), dict(window=1), dict(window=33),
                                     dict(slopes=True, softcap=50.0, window=500)])
def test_decode_torch_16_bits(options):
    gen = torch.Generator().manual_seed(9)
    lengths = [50, 1, 0, 200]
    keys, values, table = pages_for(lengths, 32, 2, 64, BF16, gen)
    if options.get("window") == 33:
        table[3, :5] = 2 ** 30  # the window of 200 tokens begins at 167
    cache = PagedCache(keys, values, table, torch.tensor(lengths, dtype=torch.int32))
    query = _rows(4, 8, 64, BF16, gen)
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.linspace(0.5, 0.01, 8)
    got = paged_decode(query, cache, **options)
    for b, n in enumerate(lengths):
        for h in range(8):
            if n == 0:
                assert not bool(got[b].any())
                continue
            k, v = (t[table[b, :-(-n // 32)].long().clamp(0, t.shape[0] - 1), h // 4]
                    .reshape(-1, 64)[:n] for t in (keys, values))
            slopes = options.get("slopes")
            want, room = attend64(query[b, h:h + 1], k, v, torch.tensor([n - 1]), 64 ** -0.5, BF16,
                                  options.get("softcap", 0.0),
                                  0.0 if slopes is None else float(slopes[h]),
                                  options.get("window", 0))
            assert_within(got[b, h:h + 1], want, room, f"{b} {h}")


# -- refusals ----------------------------------------------------------------

def _parts(**change):
    args = dict(key_codes=torch.zeros(2, 1, 16, 32, dtype=torch.uint8),
                value_codes=torch.zeros(2, 1, 16, 32, dtype=torch.uint8),
                key_scales=torch.zeros(2, 1, 16, 2, 2, dtype=F16),
                value_scales=torch.zeros(2, 1, 16, 2, 2, dtype=F16),
                block_table=torch.zeros(1, 2, dtype=torch.int32),
                lengths=torch.zeros(1, dtype=torch.int32))
    return {**args, **change}


def test_cache_refusals():
    QuantizedCache(**_parts())
    shared = torch.zeros(2, 1, 16, 32, dtype=torch.uint8)
    both = torch.zeros(2, 2, 1, 16, 2, 2, dtype=F16)
    for change in (
            dict(key_codes=torch.zeros(2, 1, 16, 31, dtype=torch.uint8)),
            dict(key_codes=shared, value_codes=shared),
            dict(key_scales=both[0], value_scales=both[0]),
            dict(key_codes=torch.zeros(2, 1, 16, 64, dtype=torch.uint8)[..., ::2]),
            dict(value_codes=torch.zeros(2, 1, 32, 32, dtype=torch.uint8)),
            dict(key_scales=torch.zeros(2, 1, 16, 1, 2, dtype=F16)),
            dict(key_codes=torch.zeros(2, 1, 24, 32, dtype=torch.uint8),
                 value_codes=torch.zeros(2, 1, 24, 32, dtype=torch.uint8)),
            dict(block_table=torch.zeros(1, 2)), dict(lengths=torch.zeros(2, dtype=torch.int32)),
            dict(block_table=torch.zeros(1, 0, dtype=torch.int32))):
        with pytest.raises(ValueError):
            QuantizedCache(**_parts(**change))
    for change in (dict(key_codes=shared.int()), dict(key_scales=both[0].float()),
                   dict(dtype=torch.float32)):
        with pytest.raises(TypeError):
            QuantizedCache(**_parts(**change))
    for dim in (20, 288):
        with pytest.raises(ValueError):
            QuantizedCache.empty(2, 1, 16, dim, 1, 1)
    parts = _parts()
    with pytest.raises(ValueError):  # codes of one a byte are asked for
        QuantizedCache.packed(parts["key_codes"][..., :20], parts["value_codes"],
                              parts["key_scales"], parts["value_scales"], parts["block_table"],
                              parts["lengths"])


def test_call_refusals():
    cache = QuantizedCache.empty(4, 2, 16, 64, 3, 2)
    rows = torch.zeros(3, 2, 64, dtype=BF16)
    rotary = Rotary(RotaryConfig(head_dim=64))
    for change in (dict(key=rows.half()), dict(value=rows[:2]), dict(key=rows[:, :1]),
                   dict(query=rows), dict(rotary=Rotary(RotaryConfig(head_dim=32))),
                   dict(token_starts=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            paged_append(**{**dict(key=rows, value=rows, cache=cache), **change})
    with pytest.raises(RuntimeError):
        paged_append(rows, rows, cache, query=rows, rotary=rotary, backend="hip")
    for tokens, starts in ((2, None), (-1, None), (True, None), (3.0, None),
                           (3, torch.zeros(4)), (3, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            paged_read(cache, tokens, token_starts=starts)
    query = torch.zeros(3, 4, 64, dtype=BF16)
    for options in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=math.inf), dict(softcap=1e-40),
                    dict(softcap=math.nan), dict(window=0), dict(window=2.0), dict(window=True),
                    dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4).double()),
                    dict(slopes=torch.zeros(8)[::2]), dict(output=query[:2]),
                    dict(output=query)):
        with pytest.raises(ValueError):
            paged_decode(query, cache, **options)
    with pytest.raises(ValueError):
        paged_decode(query[:, :3], cache)
    assert not bool(paged_decode(query, cache).any())  # every place is idle


def test_rows_in_the_cache_are_refused():
    cache = QuantizedCache.empty(16, 2, 16, 64, 3, 2)
    inside = cache.key_codes.view(-1).view(BF16)[:384].view(3, 2, 64)
    rows = torch.zeros(3, 2, 64, dtype=BF16)
    for change in (dict(key=inside), dict(value=inside),
                   dict(query=inside, rotary=Rotary(RotaryConfig(head_dim=64)))):
        with pytest.raises(ValueError, match="overlap the cache"):
            paged_append(**{**dict(key=rows, value=rows, cache=cache), **change})
