"""Prompts' attention in 64 bits, one head at a time, for its tests."""

import torch

from paged_math import assert_within
from quantized_math import attend64


def prompt64(query, key, value, starts, key_starts, scaling=None, softcap=0.0, slopes=None,
             window=0, prefix=None):
    """((tokens, q_heads, dim) outputs, error bound); rows of no sequence zeros.
    Weights enter the second product rounded to the rows' type."""
    _, q_heads, dim = query.shape
    heads = key.shape[1]
    group = q_heads // heads
    scaling = dim ** -0.5 if scaling is None else scaling
    out = torch.zeros(query.shape, dtype=torch.float64)
    room = torch.zeros(query.shape, dtype=torch.float64)
    weight_room = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(query.dtype, 0.0)
    for b in range(len(starts) - 1):
        first, end = int(starts[b]), int(starts[b + 1])
        k0, k1 = int(key_starts[b]), int(key_starts[b + 1])
        if first >= end:
            continue
        position = k1 - k0 - end + torch.arange(first, end)
        seen = 0 if prefix is None else min(max(int(prefix[b]), 0), k1 - k0)
        for h in range(q_heads):
            k, v = (t[k0:k1, h // group] for t in (key, value))
            live = position >= 0
            if k1 == k0 or not bool(live.any()):
                continue
            rows = torch.arange(first, end)[live]
            out[rows, h], room[rows, h] = attend64(
                query[rows, h], k, v, position[live], scaling, query.dtype, softcap,
                0.0 if slopes is None else float(slopes[h]), window, seen,
                weight_room=weight_room)
    return out, room


def assert_rows(got, want, room, what=""):
    """assert_within, and infinities where they are."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(got.isinf(), want.isinf()), f"{what}: infinite where it should not be, or not"
    assert torch.equal(got[got.isinf()], want[want.isinf()]), what
    finite = ~want.isinf()
    assert_within(got.where(finite, 0.0), want.where(finite, 0.0), room.where(finite, 0.0), what)
