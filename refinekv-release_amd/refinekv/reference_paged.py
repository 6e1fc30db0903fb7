"""torch restatement of the rotary and paged-cache operators
(``backend="torch"``, CPU tensors, and on a GPU the types and shapes the
kernels do not take): angles in 64 bits, products and sums in 32 (64 for
float64 inputs), one rounding at the end."""

import math

import torch


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def rotate(x, positions, rotary, inverse=False, live=None):
    """(tokens, heads, dim) rows turned to their positions; rows where
    ``live`` is false pass."""
    half = rotary.turns.numel()
    turns = positions.double()[:, None] * rotary.turns
    angles = (turns - turns.round()) * (2 * math.pi)
    wide = _wide(x)
    c = (angles.cos().to(wide.dtype) * rotary.scale)[:, None]
    s = (angles.sin().to(wide.dtype) * (-rotary.scale if inverse else rotary.scale))[:, None]
    if rotary.config.interleaved:
        first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    else:
        first, second = slice(0, half), slice(half, 2 * half)
    a, b = wide[..., first], wide[..., second]
    y = x.clone(memory_format=torch.contiguous_format)
    y[..., first] = (a * c - b * s).to(x.dtype)
    y[..., second] = (b * c + a * s).to(x.dtype)
    return y if live is None else torch.where(live[:, None, None], y, x)


def append(cache, key, value, query, rotary, token_starts):
    """paged_append's rows; returns the turned query or None."""
    tokens = key.shape[0]
    token = torch.arange(tokens, device=key.device)
    lengths = cache.lengths.long()
    if token_starts is None:
        sequence, live = token, torch.ones_like(token, dtype=torch.bool)
        position = lengths - 1
    else:
        starts = token_starts.long()
        sequence = torch.searchsorted(starts[1:].contiguous(), token, right=True)
        live = sequence < cache.sequences
        sequence = sequence.clamp_max(cache.sequences - 1)
        live &= token >= starts[sequence]
        position = lengths[sequence] - starts[sequence + 1] + token
    live = live & (position >= 0)
    position = position.clamp_min(0)
    block = position // cache.page_size
    page = cache.block_table[sequence, block.clamp_max(cache.max_blocks - 1)].long()
    stored = live & (block < cache.max_blocks) & (page >= 0) & (page < cache.pages)
    turned = key if rotary is None else rotate(key, position, rotary)
    at, row = page[stored], (position % cache.page_size)[stored]
    # (all rows are read before any is stored: they may be views of the pages)
    out = None if query is None else rotate(query, position, rotary, live=live)
    turned, value = turned[stored], value[stored]
    cache.keys[at, :, row] = turned
    cache.values[at, :, row] = value
    return out


def decode(query, cache, scaling):
    heads, dim = cache.heads, cache.head_dim
    group = query.shape[1] // heads
    out = torch.zeros(query.shape, dtype=query.dtype, device=query.device)
    for b, length in enumerate(cache.lengths.tolist()):
        if length <= 0:
            continue
        pages = cache.block_table[b, :-(-length // cache.page_size)].long()
        if length > cache.capacity or not bool(((pages >= 0) & (pages < cache.pages)).all()):
            out[b] = math.nan
            continue
        # (blocks, heads, page, dim) -> (heads, length, dim)
        k, v = (_wide(x[pages].transpose(0, 1).reshape(heads, -1, dim)[:, :length])
                for x in (cache.keys, cache.values))
        q = _wide(query[b].reshape(heads, group, dim))
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) * scaling, -1)
        out[b] = torch.matmul(p, v).reshape(heads * group, dim).to(query.dtype)
    return out
