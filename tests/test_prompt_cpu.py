"""Prompts' attention on the CPU: the torch restatement against the same in 64
bits, and the refusals."""

import math

import pytest
import torch

from paged_math import pages_for
from prompt_math import assert_rows, prompt64
from refinekv import (PagedCache, QuantizedCache, paged_append, paged_decode, paged_prompt,
                      paged_read, prompt_attention)

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ragged(counts, heads, group, dim, dtype, gen, behind=2):
    tokens = sum(counts) + behind
    starts = torch.tensor([0] + list(counts)).cumsum(0).int()
    rows = [torch.randn(tokens, n, dim, generator=gen).to(dtype)
            for n in (heads * group, heads, heads)]
    return starts, *rows


@pytest.mark.parametrize("options", [
    {}, dict(window=5), dict(softcap=3.0, prefix=[4, 0, 100, 7]), dict(slopes=True),
    dict(slopes=True, window=3, prefix=[9, 9, 9, 9])])
@pytest.mark.parametrize("dim,dtype", [(32, BF16), (64, F16), (24, F32)])
def test_rows_torch(dim, dtype, options):
    gen = torch.Generator().manual_seed(dim)
    counts = [13, 0, 1, 30]
    starts, query, key, value = ragged(counts, 2, 3, dim, dtype, gen)
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.linspace(0.5, 0.01, 6)
    if "prefix" in options:
        options["prefix"] = torch.tensor(options["prefix"], dtype=torch.int32)
    got = prompt_attention(query, key, value, token_starts=starts, **options)
    want, room = prompt64(query, key, value, starts, starts, **options)
    assert_rows(got, want, room)
    kept = torch.full_like(query, 7.0)
    out = prompt_attention(query, key, value, token_starts=starts, output=kept, **options)
    assert out is kept and torch.equal(out[:-2], got[:-2]) and bool((out[-2:] == 7.0).all())


def test_one_sequence_and_key_starts():
    gen = torch.Generator().manual_seed(1)
    _, query, key, value = ragged([40], 1, 2, 64, BF16, gen, behind=0)
    whole = prompt_attention(query, key, value)
    starts = torch.tensor([0, 40], dtype=torch.int32)
    assert torch.equal(whole, prompt_attention(query, key, value, token_starts=starts))
    # the last rows alone, over the same keys; more rows than keys see nothing
    last = prompt_attention(query[30:], key, value, token_starts=torch.tensor([0, 10]).int(),
                            key_starts=starts)
    assert torch.equal(last, whole[30:])
    more = prompt_attention(query, key[:35], value[:35], token_starts=starts,
                            key_starts=torch.tensor([0, 35]).int())
    assert not bool(more[:5].any()) and bool(more[5:].any())


def test_infinite_and_nan_values_torch():
    gen = torch.Generator().manual_seed(2)
    starts, query, key, value = ragged([20], 1, 1, 32, BF16, gen, behind=0)
    value[6, 0, 3], value[9, 0, 4], value[12, 0, 3] = math.inf, math.nan, -math.inf
    key[15, 0, 0] = math.nan
    got = prompt_attention(query, key, value, token_starts=starts)
    want, room = prompt64(query, key, value, starts, starts)
    assert_rows(got, want, room)
    assert bool(got[:6].isfinite().all()) and bool(got[15:].isnan().all())


@pytest.mark.parametrize("options", [{}, dict(window=20, softcap=5.0)])
def test_pages_torch(options):
    gen = torch.Generator().manual_seed(3)
    lengths, counts = [40, 0, 33, 7], [12, 0, 33, 3]
    keys, values, table = pages_for(lengths, 16, 2, 32, F16, gen)
    table[0, 0] = 1 << 20  # tokens 0..15 of the first sequence: gone
    cache = PagedCache(keys, values, table, torch.tensor(lengths, dtype=torch.int32))
    starts = torch.tensor([0] + counts).cumsum(0).int()
    query = torch.randn(50, 4, 32, generator=gen).to(F16)
    got = paged_prompt(query, cache, token_starts=starts, **options)
    assert not bool(got[48:].any())
    if not options:
        assert bool(got[:12].isnan().all())
    else:  # rows from 28 on see tokens from 9 on at least: 35 is the first past 15
        assert bool(got[:7].isnan().all()) and bool(got[7:].isfinite().all())
    key, value = paged_read(cache, 48, token_starts=torch.tensor([0, 12, 12, 45, 48]).int())
    alone = prompt_attention(query[12:45], key[12:45], value[12:45], **options)
    assert torch.equal(got[12:45], alone)
    last = paged_prompt(query[:4], cache, **options)
    want = paged_decode(query[:4], cache, **options)
    assert torch.allclose(last.float(), want.float(), rtol=2e-3, atol=1e-4, equal_nan=True)


def test_pages_in_4_bits_torch():
    gen = torch.Generator().manual_seed(4)
    cache = QuantizedCache.empty(4, 2, 16, 64, 1, 3)
    cache.block_table.copy_(torch.tensor([[3, 0, 2]]))
    cache.lengths.fill_(45)
    starts = torch.tensor([0, 45], dtype=torch.int32)
    query = torch.randn(45, 4, 64, generator=gen).to(BF16)
    key, value = (torch.randn(45, 2, 64, generator=gen).to(BF16) for _ in range(2))
    paged_append(key, value, cache, token_starts=starts)
    got = paged_prompt(query, cache, token_starts=starts)
    read = [t.float() for t in paged_read(cache, 45, token_starts=starts)]
    want = prompt_attention(query.float(), *read, token_starts=starts)
    # read rows are rounded to bf16, 2^-8 of them at most
    assert float((got.float() - want).abs().max()) <= 6 * 2.0 ** -8 * float(read[1].abs().max())


def test_refusals():
    q, k = torch.zeros(6, 4, 32, dtype=BF16), torch.zeros(6, 2, 32, dtype=BF16)
    starts = torch.tensor([0, 2, 6], dtype=torch.int32)
    base = dict(query=q, key=k, value=k.clone(), token_starts=starts)
    prompt_attention(**base)
    bad = [dict(query=q[0]), dict(query=q[:, :3]), dict(query=torch.zeros(6, 4, 64, dtype=BF16)),
           dict(key=k[:5]), dict(key=k[:5], value=k[:5]), dict(value=k.half()),
           dict(key=torch.zeros(6, 0, 32, dtype=BF16)), dict(token_starts=starts.long()),
           dict(token_starts=starts[:0]), dict(token_starts=torch.zeros(6).int()[::2]),
           dict(key_starts=starts[:2]), dict(token_starts=None, key_starts=starts),
           dict(prefix=starts), dict(prefix=torch.zeros(2)), dict(window=0), dict(softcap=-2.0),
           dict(slopes=torch.zeros(2)), dict(output=q), dict(output=q[:5].clone()),
           dict(output=q.float()), dict(output=q.transpose(0, 1)), dict(backend="cuda")]
    for change in bad:
        with pytest.raises(ValueError):
            prompt_attention(**{**base, **change})
    with pytest.raises(TypeError):
        prompt_attention(*(t.int() for t in (q, k, k)))
    with pytest.raises(RuntimeError):
        prompt_attention(**base, backend="hip")
    rows = torch.zeros(8, 4, 32, dtype=BF16)
    with pytest.raises(ValueError):  # output over the keys
        prompt_attention(rows[:6], rows[2:, :2], rows[2:, 2:], output=rows[2:])
    cache = PagedCache.empty(4, 2, 16, 32, 2, 2)
    paged_prompt(q[:2], cache)
    for change in (dict(query=q), dict(query=q[:2].half()), dict(query=q[:2, :3]),
                   dict(token_starts=starts[:2]), dict(prefix=starts), dict(output=q[:2]),
                   dict(window=-1)):
        with pytest.raises(ValueError):
            paged_prompt(**{**dict(query=q[:2], cache=cache), **change})
    with pytest.raises(ValueError):  # output among the pages
        paged_prompt(q[:2], cache, output=cache.keys.view(-1)[:256].view(2, 4, 32))
