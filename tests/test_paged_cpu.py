"""Rotary positions and the paged cache on the CPU: the torch restatement
against the same in 64 bits, the scalings' closed forms, and the refusals."""

import math

import pytest
import torch

from paged_math import assert_within, decode64, pages_for, rotate64
from refinekv import (PagedCache, Rotary, RotaryConfig, paged_append, paged_decode, rotate_heads)
from refinekv.rotary import check_out, rows_overlap

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# -- the rates ---------------------------------------------------------------

def test_rates_closed_forms():
    plain = RotaryConfig(head_dim=64, base=10000.0).rates()
    assert plain[0] == 1.0 and math.isclose(plain[16], 0.01, rel_tol=1e-14)
    linear = RotaryConfig(head_dim=64, scaling="linear", factor=4.0).rates()
    assert all(math.isclose(a * 4, b, rel_tol=1e-15) for a, b in zip(linear, plain))
    # ntk: the first pair as it was, the last slowed by the whole factor
    ntk = RotaryConfig(head_dim=64, scaling="ntk", factor=8.0).rates()
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 8, plain[-1], rel_tol=1e-12)
    part = RotaryConfig(head_dim=64, rotary_dim=16)
    assert len(part.rates()) == 8 and RotaryConfig(head_dim=64).rotary_dim == 64


def test_rates_llama3_bands():
    config = RotaryConfig(head_dim=128, base=500000.0, scaling="llama3", factor=8.0,
                          original_length=8192)
    plain = RotaryConfig(head_dim=128, base=500000.0).rates()
    for rate, was in zip(config.rates(), plain):
        wave = 2 * math.pi / was
        if wave < 8192 / 4:
            assert rate == was
        elif wave > 8192:
            assert math.isclose(rate, was / 8, rel_tol=1e-14)
        else:
            assert was / 8 < rate < was
    assert config.output_scale == 1.0


def test_rates_yarn_ramp_and_factor():
    config = RotaryConfig(head_dim=128, base=1000000.0, scaling="yarn", factor=4.0,
                          original_length=32768)
    plain = RotaryConfig(head_dim=128, base=1000000.0).rates()
    shares = [(r / p - 0.25) / 0.75 for r, p in zip(config.rates(), plain)]
    # pairs 0..23 turn 32 times in 32768 positions, pairs from 40 on less than once
    low = math.floor(128 * math.log(32768 / (64 * math.pi)) / (2 * math.log(1e6)))
    high = math.ceil(128 * math.log(32768 / (2 * math.pi)) / (2 * math.log(1e6)))
    for i, share in enumerate(shares):
        want = 1 - min(max((i - low) / (high - low), 0), 1)
        assert math.isclose(share, want, abs_tol=1e-12), i
    assert math.isclose(config.output_scale, 1 + 0.1 * math.log(4.0))
    assert RotaryConfig(head_dim=128, scaling="yarn", factor=4.0,
                        attention_factor=1.0).output_scale == 1.0


def test_rates_of_the_models_match_transformers():
    """The benchmark's two model configurations, against the installed
    Transformers' own fp32 rates."""
    from transformers import LlamaConfig, Qwen2Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    yarn = Qwen2Config(hidden_size=3584, num_attention_heads=28, num_key_value_heads=4,
                       max_position_embeddings=4 * 32768,
                       rope_parameters={"rope_type": "yarn", "factor": 4.0,
                                        "original_max_position_embeddings": 32768,
                                        "rope_theta": 1000000.0})
    rates, scale = ROPE_INIT_FUNCTIONS["yarn"](yarn, "cpu")
    ours = RotaryConfig(head_dim=128, base=1000000.0, scaling="yarn", factor=4.0,
                        original_length=32768)
    assert torch.allclose(torch.tensor(ours.rates()), rates.float(), rtol=2e-6, atol=0)
    assert math.isclose(ours.output_scale, scale, rel_tol=1e-6)
    llama = LlamaConfig(hidden_size=4096, num_attention_heads=32, num_key_value_heads=8,
                        rope_parameters={"rope_type": "llama3", "factor": 8.0,
                                         "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                         "original_max_position_embeddings": 8192,
                                         "rope_theta": 500000.0})
    rates, _ = ROPE_INIT_FUNCTIONS["llama3"](llama, "cpu")
    ours = RotaryConfig(head_dim=128, base=500000.0, scaling="llama3", factor=8.0)
    assert torch.allclose(torch.tensor(ours.rates()), rates.float(), rtol=2e-6, atol=0)


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=0), dict(head_dim=64, rotary_dim=3), dict(head_dim=64, rotary_dim=66),
    dict(head_dim=64, rotary_dim=0), dict(head_dim=64, rotary_dim=True), dict(head_dim=64.0),
    dict(head_dim=64, base=1.0), dict(head_dim=64, base=math.inf), dict(head_dim=63),
    dict(head_dim=64, scaling="dynamic"), dict(head_dim=64, factor=0.5),
    dict(head_dim=64, factor=math.nan), dict(head_dim=64, original_length=0),
    dict(head_dim=64, low_freq_factor=4.0), dict(head_dim=64, beta_slow=0.0),
    dict(head_dim=64, attention_factor=0.0), dict(head_dim=64, rotary_dim=2, scaling="ntk"),
])
def test_config_refusals(kwargs):
    with pytest.raises(ValueError):
        RotaryConfig(**kwargs)


def test_rotary_takes_a_models_own_rates():
    config = RotaryConfig(head_dim=8, rotary_dim=4)
    rotary = Rotary(config, rates=torch.tensor([0.5, 0.25]))
    assert rotary.turns.dtype == torch.float64
    assert torch.allclose(rotary.turns * 2 * math.pi, torch.tensor([0.5, 0.25]).double())
    with pytest.raises(ValueError):
        Rotary(config, rates=[1.0])
    with pytest.raises(TypeError):
        Rotary(dict(head_dim=8))


# -- rotate_heads ------------------------------------------------------------

@pytest.mark.parametrize("dim,rotary_dim,interleaved,dtype", [
    (64, 64, False, BF16), (64, 16, True, F16), (7, 6, False, F32), (2, 2, True, F32)])
def test_rotate_heads_torch(dim, rotary_dim, interleaved, dtype):
    gen = torch.Generator().manual_seed(dim)
    query, key = (torch.randn(9, n, dim, generator=gen).to(dtype) for n in (4, 1))
    positions = torch.randint(-100, 131072, (9,), generator=gen)
    config = RotaryConfig(head_dim=dim, rotary_dim=rotary_dim, interleaved=interleaved,
                          scaling="yarn", factor=2.0)
    for inverse in (False, True):
        got = rotate_heads(query, key, positions, Rotary(config), inverse=inverse)
        for y, x in zip(got, (query, key)):
            want, room = rotate64(x, positions, config.rates(), config.output_scale, interleaved,
                                  inverse)
            assert_within(y, want, room)
    # in place
    again = query.clone()
    out, none = rotate_heads(again, None, positions, Rotary(config), query_out=again,
                             inverse=True)
    assert out is again and none is None and torch.equal(again, got[0])


def test_rotate_heads_refusals():
    config = RotaryConfig(head_dim=8)
    rotary = Rotary(config)
    q, k, p = torch.zeros(3, 2, 8), torch.zeros(3, 1, 8), torch.arange(3)
    ok = rotate_heads(q, k, p, rotary)
    assert len(ok) == 2
    bad = [
        dict(query=q[0]), dict(query=torch.zeros(3, 2, 6)), dict(key=torch.zeros(2, 1, 8)),
        dict(key=k.half()), dict(positions=p.float()), dict(positions=p[:2]),
        dict(positions=p[:, None]), dict(query_out=torch.zeros(3, 2, 8).half()),
        dict(query_out=torch.zeros(3, 1, 8)), dict(query_out=torch.zeros(1, 2, 8).expand(3, 2, 8)),
        dict(key=None, key_out=k), dict(query=torch.zeros(3, 0, 8)), dict(backend="cuda"),
        dict(query_out=torch.zeros(3, 8, 2).transpose(1, 2)),
    ]
    for change in bad:
        args = dict(query=q, key=k, positions=p, rotary=rotary)
        args.update(change)
        with pytest.raises(ValueError):
            rotate_heads(args.pop("query"), args.pop("key"), args.pop("positions"),
                         args.pop("rotary"), **args)
    with pytest.raises(TypeError):
        rotate_heads(q.int(), None, p, rotary)
    with pytest.raises(RuntimeError):
        rotate_heads(q, k, p, rotary, backend="hip")
    # outputs over inputs that are not their own, and over each other
    both = torch.zeros(3, 4, 8)
    with pytest.raises(ValueError):
        rotate_heads(both[:, :2], both[:, 2:3], p, rotary, query_out=both[:, 1:3])
    with pytest.raises(ValueError):
        rotate_heads(q, k, p, rotary, query_out=both[:, :2], key_out=both[:, 1:2])
    rotate_heads(both[:, :2], both[:, 2:3], p, rotary, query_out=both[:, :2],
                 key_out=both[:, 2:3])


def test_rows_overlap_knows_columns_of_one_matrix():
    m = torch.zeros(10, 6, 8)
    assert not rows_overlap(m[:, :2], m[:, 2:5]) and not rows_overlap(m[:, 4:], m[:, :4])
    assert rows_overlap(m[:, :3], m[:, 2:5]) and rows_overlap(m, m)
    assert not rows_overlap(m[:5], m[5:]) and rows_overlap(m[:6], m[5:])
    # columns that start in another row are still columns
    assert not rows_overlap(m[1:, :2], m[:, 2:5])
    assert not rows_overlap(m[:, 2:5], m[1:, :2])
    with pytest.raises(ValueError):
        check_out("out", m.as_strided((10, 2, 8), (8, 8, 1)), m[:, :2])


# -- the cache ---------------------------------------------------------------

def _case(lengths, page=16, heads=2, group=3, dim=32, dtype=BF16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    keys, values, table = pages_for(lengths, page, heads, dim, dtype, gen)
    query = torch.randn(len(lengths), heads * group, dim, generator=gen).to(dtype)
    return query, keys, values, table, torch.tensor(lengths, dtype=torch.int32)


@pytest.mark.parametrize("lengths,dtype", [([1, 0, 16, 17, 70], BF16), ([5], F16), ([0], BF16)])
def test_decode_torch(lengths, dtype):
    query, *cache = _case(lengths, dtype=dtype)
    got = paged_decode(query, PagedCache(*cache))
    want, room = decode64(query, *cache, 32 ** -0.5)
    assert_within(got, want, room + 2.0 ** -12 * want.abs().nan_to_num())
    out = torch.empty_like(query)
    assert paged_decode(query, PagedCache(*cache), output=out) is out and torch.equal(out, got)


def test_decode_torch_bad_pages_and_lengths():
    query, keys, values, table, lengths = _case([20, 20, 20, 20])
    table[0, 1], table[1, 0] = -1, keys.shape[0]
    lengths[2] = table.shape[1] * 16 + 1
    got = paged_decode(query, PagedCache(keys, values, table, lengths))
    assert got[:3].isnan().all() and not got[3].isnan().any()


def test_append_torch_places_every_row():
    gen = torch.Generator().manual_seed(2)
    lengths, new, page, heads, dim = [20, 0, 3, 33], [7, 0, 5, 1], 16, 2, 8
    keys, values, table = pages_for(lengths, page, heads, dim, F32, gen)
    starts = torch.tensor([0, 7, 7, 12, 13], dtype=torch.int32)
    total = 13 + 4  # rows behind the last sequence
    key, value, query = (torch.randn(total, n, dim, generator=gen) for n in (heads, heads, 6))
    cache = PagedCache(keys.clone(), values.clone(), table,
                       torch.tensor(lengths, dtype=torch.int32))
    config = RotaryConfig(head_dim=dim, rotary_dim=4, interleaved=True)
    out = paged_append(key, value, cache, query=query, rotary=Rotary(config), token_starts=starts)
    positions, live = torch.zeros(total, dtype=torch.long), torch.zeros(total, dtype=torch.bool)
    for b in range(4):
        for j in range(new[b]):
            t = int(starts[b]) + j
            p = lengths[b] - new[b] + j
            if p >= 0:
                positions[t], live[t] = p, True
    assert live.sum() == 7 + 3 + 1  # two of sequence 2's five have no place
    want, room = rotate64(query, positions, config.rates(), interleaved=True)
    assert_within(out[live], want[live], room[live])
    assert torch.equal(out[~live], query[~live])
    want, room = rotate64(key, positions, config.rates(), interleaved=True)
    touched = torch.zeros(keys.shape[0], page, dtype=torch.bool)
    for t in live.nonzero()[:, 0].tolist():
        b = int((starts[1:] <= t).sum())
        at, row = int(table[b, positions[t] // page]), int(positions[t]) % page
        touched[at, row] = True
        assert_within(cache.keys[at, :, row], want[t], room[t])
        assert torch.equal(cache.values[at, :, row], value[t])
    rest = ~touched[:, None, :, None].expand_as(keys)
    for new_t, old in ((cache.keys, keys), (cache.values, values)):
        assert torch.equal(new_t[rest].view(torch.int32), old[rest].view(torch.int32))


def test_append_torch_no_tokens():
    cache = PagedCache.empty(4, 2, 16, 8, 3, 2, dtype=F32)
    rows = torch.empty(0, 2, 8)
    out = paged_append(rows, rows, cache, query=rows, rotary=Rotary(RotaryConfig(head_dim=8)),
                       token_starts=torch.zeros(4, dtype=torch.int32))
    assert out.shape == (0, 2, 8)


def test_cache_refusals():
    _, keys, values, table, lengths = _case([20, 20])
    PagedCache(keys, values, table, lengths)
    bad = [
        (keys[0], values[0], table, lengths), (keys, values[:, :1], table, lengths),
        (keys, values.half(), table, lengths), (keys[:, :, :12], values[:, :, :12], table, lengths),
        (keys, values, table.long(), lengths), (keys, values, table[0], lengths),
        (keys, values, table, lengths.long()), (keys, values, table, lengths[:1]),
        (keys, values, table[:, :0], lengths),
        (keys.transpose(2, 3).contiguous().transpose(2, 3), values, table, lengths),
        (keys, values, table.t().contiguous().t(), lengths),
        (keys[:, :1].expand(-1, 2, -1, -1), values, table, lengths),
        (keys, values, table, lengths.repeat_interleave(2)[::2]),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            PagedCache(*args)
    with pytest.raises(TypeError):
        PagedCache(keys.int(), values.int(), table, lengths)
    cache = PagedCache.empty(3, 2, 16, 8, 4, 5, dtype=F16)
    assert (cache.pages, cache.heads, cache.page_size, cache.head_dim) == (3, 2, 16, 8)
    assert (cache.sequences, cache.max_blocks, cache.capacity) == (4, 5, 80)
    assert (cache.block_table == -1).all() and (cache.lengths == 0).all()


def test_append_refusals():
    cache = PagedCache.empty(3, 2, 16, 8, 4, 5, dtype=F32)
    rotary = Rotary(RotaryConfig(head_dim=8))
    rows = torch.zeros(4, 2, 8)
    q, starts = torch.zeros(4, 6, 8), torch.arange(5, dtype=torch.int32)
    paged_append(rows, rows.clone(), cache, query=q, rotary=rotary, token_starts=starts)
    bad = [
        dict(key=rows[:, :1]), dict(value=rows[:3]), dict(key=rows.half()),
        dict(value=torch.zeros(4, 2, 6)), dict(token_starts=starts[:4]),
        dict(token_starts=starts.long()), dict(key=rows[:3], value=rows[:3]),
        dict(query=q), dict(rotary=Rotary(RotaryConfig(head_dim=16))),
        dict(query=q[:3], rotary=rotary), dict(query_out=q), dict(backend="none"),
        dict(query=q, rotary=rotary, query_out=torch.zeros(4, 6, 8).half()),
        dict(query=q, rotary=rotary, query_out=torch.cat([q, rows], 1)[:, 1:7].expand(4, 6, 8),
             key="inside"),
    ]
    for change in bad:
        args = dict(key=rows, value=rows.clone())
        args.update(change)
        if args["key"] is not rows and isinstance(args["key"], str):
            both = torch.zeros(4, 8, 8)
            args["key"], args["query_out"] = both[:, 6:], both[:, 1:7]
        with pytest.raises(ValueError):
            paged_append(args.pop("key"), args.pop("value"), cache, **args)
    with pytest.raises(RuntimeError):
        paged_append(rows, rows.clone(), cache, backend="hip")


def test_decode_refusals():
    query, *parts = _case([20, 20])
    cache = PagedCache(*parts)
    bad = [dict(query=query[:1]), dict(query=query[:, :5]), dict(query=query.half()),
           dict(query=query[..., :16]), dict(output=query), dict(output=query[:1].clone()),
           dict(output=query.float()), dict(backend="cuda")]
    for change in bad:
        args = dict(query=query)
        args.update(change)
        with pytest.raises(ValueError):
            paged_decode(args.pop("query"), cache, **args)
    with pytest.raises(RuntimeError):
        paged_decode(query, cache, backend="hip")


def test_c_entries_refuse_on_the_host():
    """Bad shapes, strides and pointers come back as error codes before any
    launch (the pointers below are never followed)."""
    import ctypes

    from refinekv import _hip

    lib = _hip.lib()

    def cache(**over):
        fields = dict(keys=4096, values=4096, block_table=4096, lengths=4096, pages=4, heads=2,
                      page_size=16, dim=64, sequences=2, max_blocks=3, dtype=0, table_stride=3,
                      key_strides=(ctypes.c_int64 * 3)(2048, 1024, 64),
                      value_strides=(ctypes.c_int64 * 3)(2048, 1024, 64))
        fields.update(over)
        return _hip._PagedCache(**fields)

    def decode(view, query=4096, stride=512, group=4, out=4096, workspace=4096, nbytes=1 << 40):
        return lib.rkv_paged_decode(ctypes.byref(view), query, stride, 64, group, 0.125, out,
                                    workspace, nbytes, None)

    def append(view, tokens=2, starts=None, rates=4096, rotary_dim=64, key=4096, q_heads=0):
        return lib.rkv_paged_append(ctypes.byref(view), None, 0, 0, q_heads, None, 0, 0, key, 128,
                                    64, 4096, 128, 64, tokens, starts, rates, rotary_dim, 0, 1.0,
                                    None)

    for view, code in [
            (cache(keys=None), 1), (cache(lengths=None), 1), (cache(pages=0), 1),
            (cache(sequences=0), 1), (cache(max_blocks=1 << 28), 1), (cache(page_size=24), 2),
            (cache(dtype=7), 2), (cache(table_stride=-1), 1)]:
        assert decode(view) == code and append(view) == code, lib.rkv_last_error()
    odd = (ctypes.c_int64 * 3)(2048, 1024, 60)
    for got, code in [
            (decode(cache(dtype=2)), 2), (decode(cache(dim=48)), 2), (decode(cache(dim=288)), 2),
            (decode(cache(), group=17), 2), (decode(cache(), group=0), 1),
            (decode(cache(key_strides=odd)), 1), (decode(cache(values=4104)), 1),
            (decode(cache(), query=None), 1), (decode(cache(), query=4098), 1),
            (decode(cache(), stride=513), 1), (decode(cache(), out=None), 1),
            (append(cache(), tokens=3), 1), (append(cache(), tokens=-1, starts=4096), 1),
            (append(cache(), rotary_dim=3), 1), (append(cache(), rotary_dim=66), 1),
            (append(cache(), rates=None), 1), (append(cache(), key=None), 1),
            (append(cache(), key=4097), 1), (append(cache(), q_heads=4), 1)]:
        assert got == code, lib.rkv_last_error()
    assert lib.rkv_paged_decode(None, 4096, 512, 64, 4, 0.1, 4096, 4096, 0, None) == 1
    assert lib.rkv_rotary(None, 0, 0, 2, None, 0, 0, 0, 0, 5, 64, 4096, 1, 4096, 64, 0, 1.0, 0,
                          None, 0, 0, None, 0, 0, None) == 1
    assert lib.rkv_rotary(4096, 0, 0, 2, None, 0, 0, 0, 9, 5, 64, 4096, 1, 4096, 64, 0, 1.0, 0,
                          4096, 0, 0, None, 0, 0, None) == 2
