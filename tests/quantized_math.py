"""The paged cache in 4 bits and the scores' options in 64 bits, for their tests.

Written from the definitions, on the CPU, one sequence and head at a time, apart
from the package's own torch operations; bounds count the roundings of a 32-bit
computation as paged_math's do.
"""

import math

import numpy as np
import torch

from paged_math import half_step, tiny


def scale64(span):
    """A 15th of the span as the nearest fp16 number, then rounded up to 7
    significant bits (steps of 2^-20 below 2^-14)."""
    near = np.float16(np.float32(span) / np.float32(15.0)).astype(np.float64)
    _, e = np.frexp(np.maximum(near, 2.0 ** -14))
    unit = 2.0 ** (e - 7.0)
    return np.ceil(near / unit) * unit


def quantize64(rows):
    """((.., dim) codes, scales and zeros per dim) of rows, as float64 arrays;
    NaN scales and zeros where a group is not held."""
    x = rows.double().numpy()
    groups = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        held = np.isfinite(groups).all(-1) & (np.abs(groups).max(-1) <= 4096.0)
        safe = np.where(held[..., None], groups, 0.0)
        zero = safe.min(-1).astype(np.float16).astype(np.float64)
        # (in fp32, as a span of two 16-bit numbers need not be one)
        span = safe.max(-1).astype(np.float32) - safe.min(-1).astype(np.float32)
        scale = scale64(span)
        codes = np.rint(((safe - zero[..., None]).astype(np.float32)
                         / scale[..., None].astype(np.float32)).astype(np.float64))
        codes = np.where(scale[..., None] > 0, np.clip(codes, 0, 15), 0.0)
    scale, zero = (np.where(held, t, np.nan) for t in (scale, zero))
    wide = [np.repeat(t[..., None], 32, -1).reshape(x.shape) for t in (scale, zero)]
    return codes.reshape(x.shape), *wide


def attend64(q, k, v, position, scaling, dtype, softcap=0.0, slope=0.0, window=0, prefix=0,
             size=None, weight_room=2.0 ** -16, value_size=None):
    """(rows, dim) outputs of one head's query rows at their positions, and how
    far a correct 32-bit computation may be off.

    ``size`` (rows, tokens): sums of the magnitudes that a score is summed from
    (|q| |k| unless given), whose order of summation is free; ``weight_room``:
    what a weight is rounded by on its way into the second product;
    ``value_size``: magnitudes that the outputs are summed from."""
    q, k, v = q.double(), k.double(), v.double()
    dim, n = q.shape[1], k.shape[0]
    token = torch.arange(n)
    distance = position[:, None] - token
    seen = (distance >= 0) | (token < prefix)
    if window:
        seen &= distance < window
    x = q @ k.T * scaling
    size = (q.abs() @ k.abs().T if size is None else size) * abs(scaling)
    room = (dim + 6) * 2.0 ** -24 * size
    if softcap:
        x = softcap * torch.tanh(x / softcap)
        room = room + softcap * 2.0 ** -22
    if slope:
        bias = slope * distance.abs()
        x = x - bias
        room = room + (3 * bias.abs() + size) * 2.0 ** -24
    live = seen.any(1)
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1)
    p[~live] = 0.0
    finite = v.isfinite()
    out = p @ torch.where(finite, v, 0.0)
    for value in (math.inf, -math.inf, math.nan):
        there = v.isnan() if math.isnan(value) else v == value
        out = out + torch.where((p > 0).double() @ there.double() > 0, value, 0.0)
    room = room.masked_fill(~seen, 0.0).amax(1, keepdim=True)
    spread = (x.amax(1, keepdim=True) - x.masked_fill(~seen, math.inf).amin(1, keepdim=True))
    spread = torch.where(live[:, None], spread.abs(), 0.0)
    relative = room + (spread + 2) * 2.0 ** -23 + weight_room + n * 2.0 ** -24
    sizes = torch.where(finite, v.abs(), 0.0) if value_size is None else value_size
    # (a weight far below the largest may be an fp16 subnormal: 2^-40 of it)
    room = 2 * relative * (p @ sizes) + 2.0 ** -40 * sizes.sum(0)
    room = room + half_step(dtype) * (out.nan_to_num(0, 0, 0).abs() + room) + tiny(dtype)
    return out, room


def decode64_quantized(query, codes, scales, zeros, table, lengths, scaling, softcap=0.0,
                       slopes=None, window=0):
    """paged_decode over a cache in 4 bits: ``codes``, ``scales``, ``zeros`` are
    pairs (keys, values) of (pages, heads, page, dim) float64 tensors.

    A query row enters in fp16 as a multiple of a power of two near its largest
    value: off by 2^-24 of that at most; scores are summed from q scale code and
    q zero apart.  Weights enter in one fp16 part (2^-12), two for fp16 rows."""
    batch, q_heads, dim = query.shape
    heads, page = codes[0].shape[1], codes[0].shape[2]
    group = q_heads // heads
    out = torch.zeros(query.shape, dtype=torch.float64)
    room = torch.zeros(query.shape, dtype=torch.float64)
    for b in range(batch):
        n = int(lengths[b])
        if n <= 0:
            continue
        first = max(n - window, 0) // page if window else 0
        take = table[b, first:-(-n // page)].long()
        if n > table.shape[1] * page or bool((take < 0).any()) or bool(
                (take >= codes[0].shape[0]).any()):
            out[b] = math.nan
            continue
        first *= page
        for h in range(heads):
            (ck, sk, zk), (cv, sv, zv) = (
                [t[i][take, h].reshape(-1, dim)[:n - first] for t in (codes, scales, zeros)]
                for i in (0, 1))
            for g in range(group):
                row = h * group + g
                q = query[b, row:row + 1].double()
                held = sk * ck + zk.abs()
                size = (q.abs() + (dim + 6) ** -1.0 * q.abs().max()) @ held.T
                o, r = attend64(q, sk * ck + zk, sv * cv + zv, torch.tensor([n - 1 - first]),
                                scaling, query.dtype, softcap,
                                0.0 if slopes is None else float(slopes[row]), window,
                                size=size.nan_to_num(0.0),
                                weight_room=2.0 ** -12 if query.dtype == torch.bfloat16
                                else 2.0 ** -22,
                                value_size=(sv * cv + zv.abs()).nan_to_num(0.0))
                out[b, row], room[b, row] = o[0], r[0]
    return out, room
