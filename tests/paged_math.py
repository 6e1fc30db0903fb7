"""The rotary and paged-cache operators in 64 bits, and inputs for their tests.

Written from the formulas, on the CPU, one sequence and head at a time; every
function also returns how far a correct 32-bit computation, rounded once to
``dtype``, may be from it.
"""

import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal step."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotate64(x, positions, rates, scale=1.0, interleaved=False, inverse=False):
    """((tokens, heads, dim) turned rows, error bound).  cos and sin from fp32
    series (about 3 units of 2^-24, the factor and two products 4 more): at
    most 8 * 2^-24 of |x0| + |x1|, then one rounding to x's type."""
    wide = x.double()
    out, room = wide.clone(), torch.zeros_like(wide)
    half = len(rates)
    sign = -1.0 if inverse else 1.0
    for i, rate in enumerate(rates):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = positions.double() * rate
        c, s = scale * angle.cos()[:, None], sign * scale * angle.sin()[:, None]
        out[..., p] = wide[..., p] * c - wide[..., q] * s
        out[..., q] = wide[..., q] * c + wide[..., p] * s
        size = 8 * 2.0 ** -24 * scale * (wide[..., p].abs() + wide[..., q].abs())
        room[..., p] = room[..., q] = size
    turned = room > 0
    room += torch.where(turned, half_step(x.dtype) * (out.abs() + room) + tiny(x.dtype), 0.0)
    return out, room


def decode64(query, keys, values, table, lengths, scaling):
    """((sequences, q_heads, dim) outputs, error bound) of bf16 or fp16 inputs.

    Scores are fp32 sums of dim products: off by at most (dim + 2) 2^-24
    sum |q k| scaling; e^x of a difference x adds |x| 2^-23 and 2 units; the
    weights enter the second product in two parts, 2^-16 apart at most; sums
    over a sequence's n weights add n 2^-24.  All of these are relative errors
    of the weights, and a weighted mean of v moves by at most twice the
    largest of them times the weighted mean of |v|; then one rounding."""
    batch, q_heads, dim = query.shape
    heads, page = keys.shape[1], keys.shape[2]
    group = q_heads // heads
    out = torch.zeros(query.shape, dtype=torch.float64)
    room = torch.zeros(query.shape, dtype=torch.float64)
    for b in range(batch):
        n = int(lengths[b])
        if n <= 0:
            continue
        take = table[b, :-(-n // page)].long()
        if n > table.shape[1] * page or bool((take < 0).any()) or bool(
                (take >= keys.shape[0]).any()):
            out[b] = math.nan
            continue
        for h in range(heads):
            k = keys[take, h].reshape(-1, dim)[:n].double()
            v = values[take, h].reshape(-1, dim)[:n].double()
            q = query[b, h * group:(h + 1) * group].double()
            scores = q @ k.T * scaling
            p = torch.softmax(scores, -1)
            rows = slice(h * group, (h + 1) * group)
            out[b, rows] = p @ v
            size = (q.abs() @ k.abs().T * abs(scaling)).amax(-1, keepdim=True)
            spread = (scores.amax(-1, keepdim=True) - scores).amax(-1, keepdim=True)
            relative = ((dim + 2) * 2.0 ** -24 * size + (spread + 2) * 2.0 ** -23 + 2.0 ** -16
                        + n * 2.0 ** -24)
            room[b, rows] = 2 * relative * (p @ v.abs())
    room += half_step(query.dtype) * (out.abs() + room) + tiny(query.dtype)
    return out, room


def assert_within(got, want, room, what=""):
    """got's finite values within room of want's; NaN exactly where want is."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN where there should be none, or not"
    live = ~want.isnan()
    over = ((got - want).abs() - room)[live]
    assert not over.numel() or float(over.max()) <= 0, (
        f"{what}: {float((got - want).abs()[live].max()):.3e} off, "
        f"{float(over.max()):.3e} over what rounding explains")


def pages_for(lengths, page, heads, dim, dtype, gen, spare=2, extra_blocks=1, last=0):
    """(keys, values, table): pages of randn in random order, NaN in every row
    no sequence sees (page tails included), table entries past the end that
    are out of range either way."""
    blocks = [-(-max(int(n), 0) // page) for n in lengths]
    count = sum(blocks) + spare
    order = torch.randperm(count, generator=gen)
    shape = (count, heads, page, dim)
    keys = torch.full(shape, math.nan, dtype=dtype)
    values = torch.full(shape, math.nan, dtype=dtype)
    table = torch.full((len(blocks), max(blocks) + extra_blocks), -1, dtype=torch.int32)
    table[:, -1] = 2 ** 31 - 1 if extra_blocks else table[:, -1]
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
        rows = int(lengths[b])
        for t in (keys, values):
            data = torch.randn(max(rows, 0), heads, dim, generator=gen).to(dtype)
            for j in range(n):
                part = data[j * page:(j + 1) * page].transpose(0, 1)
                t[int(table[b, j]), :, :part.shape[1]] = part
    return keys, values, table
