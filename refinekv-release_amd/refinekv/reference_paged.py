"""torch restatement of the rotary and paged-cache operators
(``backend="torch"``, CPU tensors, and on a GPU the types and shapes the
kernels do not take): angles in 64 bits, products and sums in 32 (64 for
float64 inputs), one rounding at the end."""

import math

import torch

from . import quantized
from .quantized import QuantizedCache


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


def places(cache, tokens, token_starts):
    """(position, live, stored, page) of new tokens' rows: live ones have a
    position, stored ones a page of the cache."""
    device = cache.device
    token = torch.arange(tokens, device=device)
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
    return position, live, stored, page


def append(cache, key, value, query, rotary, token_starts):
    """paged_append's rows; returns the turned query or None."""
    position, live, stored, page = places(cache, key.shape[0], token_starts)
    turned = key if rotary is None else rotate(key, position, rotary)
    at, row = page[stored], (position % cache.page_size)[stored]
    # (all rows are read before any is stored: they may be views of the pages)
    out = None if query is None else rotate(query, position, rotary, live=live)
    turned, value = turned[stored], value[stored]
    if isinstance(cache, QuantizedCache):
        pools = ((cache.key_codes, cache.key_scales, KEYS, turned),
                 (cache.value_codes, cache.value_scales, VALUES, value))
        # (a token's codes lie among its neighbours': whole pages are coded anew)
        pages, local = at.unique(return_inverse=True)
        for codes, scales, order, rows in pools:
            plain = [order[0](codes[pages]), order[1](scales[pages])]
            for pool, new in zip(plain, quantized.quantize(rows)):
                pool[local, :, row] = new
            codes[pages], scales[pages] = order[2](plain[0]), order[3](plain[1])
        return out
    cache.keys[at, :, row] = turned
    cache.values[at, :, row] = value
    return out


# unpack codes and scales, pack codes and scales
KEYS = (quantized.unpack_keys, torch.clone, quantized.pack_keys, torch.clone)
VALUES = (quantized.unpack_values, quantized.unpack_scales, quantized.pack_values,
          quantized.pack_scales)


def pages_of(cache, pages):
    """(pages, heads, page_size, head_dim) keys and values, in 32 bits or more."""
    if isinstance(cache, QuantizedCache):
        return tuple(quantized.dequantize(order[0](codes[pages]), order[1](scales[pages]))
                     for codes, scales, order in (
                         (cache.key_codes, cache.key_scales, KEYS),
                         (cache.value_codes, cache.value_scales, VALUES)))
    return _wide(cache.keys[pages]), _wide(cache.values[pages])


def read(cache, tokens, token_starts):
    """paged_read's rows."""
    position, live, stored, page = places(cache, tokens, token_starts)
    at, local = page[stored].unique(return_inverse=True)
    rows = (position % cache.page_size)[stored]
    found = []
    for pool in pages_of(cache, at):
        out = torch.zeros((tokens, cache.heads, cache.head_dim), dtype=cache.dtype,
                          device=cache.device)
        out[live & ~stored] = math.nan
        out[stored] = pool[local, :, rows].to(cache.dtype)
        found.append(out)
    return tuple(found)


def score(x, scores, distance, heads):
    """Scaled products capped and biased by the tokens' distance; ``heads``: the
    slopes' shape beside them."""
    if scores.softcap:
        x = torch.tanh(x / scores.softcap) * scores.softcap
    if scores.slopes is not None:
        x = x - scores.slopes.view(heads) * distance
    return x


def attend(q, k, v, position, scaling, scores, prefix=0):
    """(heads, group, rows, dim) outputs of query rows at their positions over
    (heads, tokens, dim) keys and values, in the inputs' type (32 bits or
    more); rows that see nothing are zeros."""
    token = torch.arange(k.shape[1], device=k.device)
    distance = position[:, None] - token
    x = torch.matmul(q, k[:, None].transpose(2, 3).contiguous()) * scaling
    seen = ((distance >= 0) | (token < prefix)) & (position >= 0)[:, None]
    if scores is not None:
        x = score(x, scores, distance.abs(), (*q.shape[:2], 1, 1))
        if scores.window:
            seen &= distance < scores.window
    p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
    p = p.masked_fill(~seen.any(-1, keepdim=True), 0.0)
    v = v[:, None]
    finite = v.isfinite()
    if bool(finite.all()):
        return torch.matmul(p, v)
    # (0 times infinity is NaN: infinities and NaN count for the rows that see them)
    out = torch.matmul(p, v.masked_fill(~finite, 0.0))
    for value in (math.inf, -math.inf, math.nan):
        there = v.isnan() if math.isnan(value) else v == value
        out = out + torch.where(torch.matmul(seen.to(v.dtype), there.to(v.dtype)) > 0, value, 0.0)
    return out


ATTENDED = 1 << 26  # scores held at a time


def _prompt(query, heads, starts, keys_of, scaling, scores, prefix, output):
    """Prompts' rows, a sequence at a time: keys_of(b) gives its (heads, tokens,
    dim) keys and values, or None where its rows are NaN."""
    tokens, q_heads, dim = query.shape
    group = q_heads // heads
    out = torch.zeros_like(query, memory_format=torch.contiguous_format) if output is None \
        else output
    if any(a > b for a, b in zip(starts, starts[1:])):
        return out
    for b in range(len(starts) - 1):
        first = min(max(starts[b], 0), tokens)
        end = min(max(starts[b + 1], first), tokens)
        if first == end:
            continue
        rows = keys_of(b)
        if rows is None:
            out[first:end] = math.nan
            continue
        k, v = rows
        n = k.shape[1]
        seen = 0 if prefix is None else min(max(int(prefix[b]), 0), n)
        together = max(1, ATTENDED // max(n * q_heads, 1))
        for row in range(first, end, together):
            take = slice(row, min(row + together, end))
            position = n - end + torch.arange(take.start, take.stop, device=query.device)
            q = _wide(query[take]).unflatten(1, (heads, group)).permute(1, 2, 0, 3)
            y = attend(q, k, v, position, scaling, scores, seen)
            out[take] = y.permute(2, 0, 1, 3).flatten(1, 2).to(query.dtype)
    return out


def prompt_rows(query, key, value, token_starts, key_starts, prefix, scaling, scores, output):
    starts = [0, query.shape[0]] if token_starts is None else token_starts.tolist()
    ends = starts if key_starts is None else key_starts.tolist()

    def keys_of(b):
        first = min(max(ends[b], 0), key.shape[0])
        end = min(max(ends[b + 1], first), key.shape[0])
        return tuple(_wide(t[first:end]).transpose(0, 1) for t in (key, value))

    return _prompt(query, key.shape[1], starts, keys_of, scaling, scores, prefix, output)


def prompt_pages(query, cache, token_starts, prefix, scaling, scores, output):
    starts = (list(range(query.shape[0] + 1)) if token_starts is None
              else token_starts.tolist())
    lengths = cache.lengths.tolist()

    def keys_of(b):
        n = max(lengths[b], 0)
        if n > cache.capacity:
            return None
        pages = cache.block_table[b, :-(-n // cache.page_size)].long()
        there = (pages >= 0) & (pages < cache.pages)
        k, v = pages_of(cache, torch.where(there, pages, 0))
        # (rows that see a page that is not there are NaN)
        k = k.masked_fill(~there[:, None, None, None], math.nan)
        v = v.masked_fill(~there[:, None, None, None], 0.0)
        return tuple(t.transpose(0, 1).flatten(1, 2)[:, :n] for t in (k, v))

    return _prompt(query, cache.heads, starts, keys_of, scaling, scores, prefix, output)


def decode(query, cache, scaling, scores=None):
    heads, dim = cache.heads, cache.head_dim
    group = query.shape[1] // heads
    out = torch.zeros(query.shape, dtype=query.dtype, device=query.device)
    for b, length in enumerate(cache.lengths.tolist()):
        if length <= 0:
            continue
        # (tokens before the window are hidden, their pages may be gone)
        hidden = 0
        if scores is not None and scores.window:
            hidden = max(length - scores.window, 0)
        first = hidden // cache.page_size
        pages = cache.block_table[b, first:-(-length // cache.page_size)].long()
        if length > cache.capacity or not bool(((pages >= 0) & (pages < cache.pages)).all()):
            out[b] = math.nan
            continue
        first *= cache.page_size
        # (blocks, heads, page, dim) -> (heads, length, dim)
        k, v = (x.transpose(0, 1).reshape(heads, -1, dim)[:, hidden - first:length - first]
                for x in pages_of(cache, pages))
        q = _wide(query[b].reshape(heads, group, dim))
        x = torch.matmul(q, k.transpose(1, 2)) * scaling
        if scores is not None:
            distance = torch.arange(k.shape[1] - 1, -1, -1, device=query.device)
            x = score(x, scores, distance, (heads, group, 1))
        p = torch.softmax(x, -1)
        out[b] = torch.matmul(p, v).reshape(heads * group, dim).to(query.dtype)
    return out
