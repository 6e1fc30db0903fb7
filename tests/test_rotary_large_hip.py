"""Rotary positions and the append at sizes where a thread turns several heads
and stores pass the caches (GPU): a sample of rows against 64 bits, and every
row against the same rows turned a few tokens at a time, bit for bit."""

import pytest
import torch

from paged_math import assert_within, rotate64
from refinekv import PagedCache, Rotary, RotaryConfig, paged_append, rotate_heads

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STREAM_BYTES = 256 << 20


def bits(t):
    return t.contiguous().view(torch.uint8)


def _in_pieces(rows, positions, rotary, piece):
    parts = [rotate_heads(rows[t:t + piece], None, positions[t:t + piece], rotary, backend="hip")[0]
             for t in range(0, len(rows), piece)]
    return torch.cat(parts)


CASES = [  # tokens, heads, KV heads, dim, rotary_dim, interleaved, dtype, passes the caches
    (5003, 17, 3, 128, 128, False, BF16, False), (14003, 17, 3, 128, 128, False, BF16, False),
    (53003, 17, 3, 128, 128, False, BF16, True), (30001, 7, 2, 256, 64, True, F32, True),
    (21011, 13, 4, 96, 48, True, F16, False), (83011, 13, 4, 96, 48, True, F16, True),
    (24007, 40, 5, 128, 64, False, BF16, True), (100003, 43, 7, 7, 6, False, F16, False),
    (390011, 43, 7, 7, 6, True, BF16, True), (106013, 9, 1, 128, 128, True, BF16, True),
    (2039, 131, 2, 256, 256, False, F32, True), (7001, 16, 3, 88, 48, True, F16, False),
]


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary_dim,interleaved,dtype,streams", CASES)
def test_rotate_heads_of_many_tokens(tokens, heads, kv, dim, rotary_dim, interleaved, dtype,
                                     streams):
    gen = torch.Generator("cuda").manual_seed(tokens + dim)
    fused = torch.randn(tokens, heads + kv + 1, dim, generator=gen, device="cuda").to(dtype)
    query, key, rest = fused[:, :heads], fused[:, heads:-1], fused[:, -1:].clone()
    positions = torch.randint(0, 131072, (tokens,), generator=gen, device="cuda")
    config = RotaryConfig(head_dim=dim, rotary_dim=rotary_dim, base=500000.0,
                          interleaved=interleaved)
    rotary = Rotary(config, "cuda")
    assert (tokens * (heads + kv) * dim * fused.element_size() >= STREAM_BYTES) == streams
    want = [_in_pieces(x, positions, rotary, 97 if tokens < 20000 else 499) for x in (query, key)]
    pick = torch.cat([torch.arange(40), torch.arange(tokens - 40, tokens),
                      torch.randint(0, tokens, (100,), generator=torch.Generator().manual_seed(1))])
    for x, y in zip((query, key), want):
        exact, room = rotate64(x[pick.cuda()].cpu(), positions[pick.cuda()].cpu(), config.rates(),
                               interleaved=interleaved)
        assert_within(y[pick.cuda()], exact, room)
    got = rotate_heads(query, key, positions, rotary, backend="hip")
    for y, x in zip(got, want):
        assert torch.equal(bits(y), bits(x))
    # over the inputs, what lies beside them left alone
    again = rotate_heads(query, key, positions, rotary, query_out=query, key_out=key, backend="hip")
    for y, x in zip(again, want):
        assert torch.equal(bits(y), bits(x))
    assert torch.equal(bits(fused[:, -1:]), bits(rest))


@pytest.mark.parametrize("tokens,heads,kv,dim,rotary_dim,interleaved,dtype,streams", CASES)
def test_append_of_many_tokens(tokens, heads, kv, dim, rotary_dim, interleaved, dtype, streams):
    """Three prompts of unequal length and some rows of none behind them."""
    gen = torch.Generator("cuda").manual_seed(tokens + dim + 1)
    query, key, value = (torch.randn(tokens, n, dim, generator=gen, device="cuda").to(dtype)
                         for n in (heads, kv, kv))
    page = 32
    lengths = [tokens // 5, tokens - tokens // 5 - 50 - 3, 50]
    starts = [0, lengths[0], lengths[0] + lengths[1], tokens - 3]
    blocks = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(blocks) + 2, generator=torch.Generator().manual_seed(2)).int()
    table = torch.full((3, max(blocks)), -1, dtype=torch.int32)
    for b, n in enumerate(blocks):
        table[b, :n] = order[sum(blocks[:b]):sum(blocks[:b]) + n]
    pages = torch.full((2, len(order), kv, page, dim), 3.0, dtype=dtype, device="cuda")
    cache = PagedCache(pages[0], pages[1], table.cuda(),
                       torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    config = RotaryConfig(head_dim=dim, rotary_dim=rotary_dim, interleaved=interleaved,
                          scaling="yarn", factor=4.0, original_length=32768)
    rotary = Rotary(config, "cuda")
    positions = torch.cat([torch.arange(n) for n in lengths]).cuda()
    turned = [_in_pieces(x[:tokens - 3], positions, rotary, 97 if tokens < 20000 else 499)
              for x in (query, key)]
    out = paged_append(key, value, cache, query=query, rotary=rotary,
                       token_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                       backend="hip")
    assert torch.equal(bits(out[:-3]), bits(turned[0]))
    assert torch.equal(bits(out[-3:]), bits(query[-3:]))
    for t, rows in zip(pages, (turned[1], value[:-3])):
        want = torch.full_like(t, 3.0)
        for b, n in enumerate(lengths):
            at = torch.arange(n)
            place = table[b, at // page].long().cuda(), (at % page).cuda()
            want[place[0], :, place[1]] = rows[starts[b]:starts[b + 1]]
        assert torch.equal(bits(t), bits(want))
