"""Infinite and NaN values that a sequence sees count as in a softmax: an
infinity whose weight is not 0 makes its dim infinite, infinities of both signs
or one of weight 0 make it NaN, and the other dims do not change."""

import math

import pytest
import torch

from paged_math import half_step, tiny
from refinekv import PagedCache, paged_decode

BF16, F16 = torch.bfloat16, torch.float16
KINDS = {"inf": math.inf, "-inf": -math.inf, "nan": math.nan}


def _case(lengths, page, heads, group, dim, dtype, seed):
    """(query, keys, values, table, lengths), the 64-bit result and its room.

    Scores are the keys' last dim, exact in the type, between -1 and 0, but for
    one of 0 early or late in a sequence, one of -40 (a weight of 2^-58) and one
    of -inf."""
    gen = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lengths]
    table = torch.full((len(lengths), max(blocks)), -1, dtype=torch.int32)
    order = torch.randperm(sum(blocks), generator=gen).int()
    shape = (sum(blocks), heads, page, dim)
    keys, values = torch.zeros(shape, dtype=dtype), torch.full(shape, math.nan, dtype=dtype)
    query = torch.zeros(len(lengths), heads * group, dim, dtype=dtype)
    query[..., -1] = 1.0
    out = torch.zeros(query.shape, dtype=torch.float64)
    room = torch.zeros(query.shape, dtype=torch.float64)
    for b, n in enumerate(lengths):
        at = sum(blocks[:b])
        table[b, :blocks[b]] = order[at:at + blocks[b]]
        score = (-torch.rand(heads, n, generator=gen)).to(dtype)
        v = torch.randn(heads, n, dim, generator=gen).to(dtype)
        for h in range(heads):
            # (places of their own, as far as the sequence has so many)
            top, far, gone, some, other = (torch.randperm(max(n, 5), generator=gen)[:5] % n).tolist()
            score[h, top] = 0.0
            if n >= 5:
                score[h, far], score[h, gone] = -40.0, -math.inf
                v[h, gone, 5] = math.inf          # times a weight of 0
                v[h, far, 2] = math.inf
                v[h, some, 3], v[h, other, 3] = math.inf, -math.inf
                v[h, some, 1] = v[h, other, 1] = -math.inf
            v[h, top, 0] = math.inf
            v[h, top, 4] = math.nan
        p = torch.softmax(score.double(), -1)[..., None]
        want = (p * v.double()).sum(1)
        # relative error of a weight: 2 units for the exponential, 3 for a score
        # of up to 40 and its difference to the maximum, and the sums' n
        relative = (2 + 3 * 40 + n) * 2.0 ** -24
        slack = 2 * relative * (p * v.double().nan_to_num(0.0, 0.0, 0.0).abs()).sum(1)
        rows = slice(0, heads * group)
        out[b, rows] = want.repeat_interleave(group, 0)
        room[b, rows] = slack.repeat_interleave(group, 0)
        for j in range(blocks[b]):
            part = slice(j * page, min((j + 1) * page, n))
            size = part.stop - part.start
            keys[int(table[b, j]), :, :size, -1] = score[:, part]
            values[int(table[b, j]), :, :size] = v[:, part]
    room += half_step(dtype) * (out.nan_to_num(0.0, 0.0, 0.0).abs() + room) + tiny(dtype)
    return (query, keys, values, table, torch.tensor(lengths, dtype=torch.int32)), out, room


def _check(got, want, room):
    got = got.cpu().double()
    for name, kind in KINDS.items():
        same = torch.tensor(kind).double()
        a, b = ((t.isnan() if name == "nan" else t == same) for t in (got, want))
        assert bool(b.any()), name
        assert torch.equal(a, b), f"{name}: {int((a != b).sum())} of {int(b.sum())} places"
    finite = want.isfinite()
    over = ((got - want).abs() - room)[finite]
    assert float(over.max()) <= 0, f"{float(over.max()):.2e} more than rounding explains"


SHAPES = [
    ([1, 5, 40, 33, 700], 16, 2, 4, 64), ([3000, 40, 2999], 32, 2, 3, 128),
    ([1500, 31, 900], 64, 1, 16, 256), ([600, 601], 16, 1, 2, 32), ([400, 77], 16, 2, 5, 96),
    ([500, 7], 32, 1, 1, 160), ([300, 90], 16, 1, 7, 192), ([257, 1200], 256, 1, 2, 224),
    ([2000 + 37 * b for b in range(7)], 16, 8, 2, 64),  # several tiles a wave
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,page,heads,group,dim", SHAPES)
def test_decode_counts_infinite_values_as_a_softmax(lengths, page, heads, group, dim, dtype):
    case, want, room = _case(lengths, page, heads, group, dim, dtype, seed=dim + len(lengths))
    query, *parts = (t.cuda() for t in case)
    _check(paged_decode(query, PagedCache(*parts), scaling=1.0, backend="hip"), want, room)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_torch_decode_counts_infinite_values_as_a_softmax(dtype):
    case, want, room = _case([1, 5, 40, 33, 700], 16, 2, 4, 64, dtype, seed=1)
    query, *parts = case
    _check(paged_decode(query, PagedCache(*parts), scaling=1.0), want, room)
