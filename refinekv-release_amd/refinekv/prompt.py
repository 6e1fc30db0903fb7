"""Attention of prompts' rows, several sequences at once.

``prompt_attention`` attends rows over the keys and values of their own
sequences, which lie one after another (documents packed into a batch; a
prompt whose cache is in 4 bits); ``paged_prompt`` attends the sequences'
last tokens over a paged cache that holds them (a prompt's chunk, the next turn
of a chat).  A row sees the tokens up to its own, all of its sequence's prefix,
and of these ``window`` back; scores may be capped and biased by distance as
``paged_decode``'s.  A layer's prompt::

    query, key = rotate_heads(query, key, positions, rotary)
    paged_append(key, value, cache, token_starts=starts)
    output = paged_prompt(query, cache, token_starts=starts)

ROCm tensors use the gfx950 kernels, others (and the types and shapes the
kernels do not take, a cache in 4 bits among them) torch operations, which read
starts and lengths on the host: those calls cannot be captured and say so.
Inference only, as the whole package: the results carry no gradient.
"""

import torch

from . import _hip
from .paged import (MAX_ROW_STRIDE, _check_capture, _check_starts, _meet_pages, check_scores)
from .quantized import QuantizedCache
from .rotary import pick_backend, rows_overlap

MOST_KEYS = 2 ** 31 - 512
HIP_DTYPES = (torch.bfloat16, torch.float16)


def _check_int32(name, t, count, device):
    if (t.shape != (count,) or t.dtype != torch.int32 or t.device != device
            or not t.is_contiguous()):
        raise ValueError(f"{name} must be contiguous int32 with shape ({count},) on the query's "
                         "device")


def _check_query(query, heads, dim):
    shape = query.shape
    if len(shape) != 3 or shape[1] <= 0 or shape[1] % heads or shape[2] != dim:
        raise ValueError("query must have shape (tokens, q_heads, head_dim) with q_heads a "
                         "multiple of the keys' heads and their head_dim")


def _check_output(output, query, others):
    if (output.shape != query.shape or output.dtype != query.dtype
            or output.device != query.device or not output.is_contiguous()):
        raise ValueError("output must be contiguous with the query's shape, dtype and device")
    if any(rows_overlap(output, t) for t in (query, *others)):
        raise ValueError("output must not overlap the query, keys or values")


def _why_not_rows(dtype, dim):
    if dtype not in HIP_DTYPES:
        return "the HIP prompt attention needs bf16 or fp16 rows"
    if dim not in _hip.SUPPORTED_DIMS:
        return "the HIP prompt attention needs head_dim in 32..256 (multiple of 32)"
    return None


def _why_not_cache(cache):
    if isinstance(cache, QuantizedCache):
        return "the HIP prompt attention needs a 16-bit cache (read a 4-bit one's rows first)"
    why = _why_not_rows(cache.dtype, cache.head_dim)
    if why is None:
        for t in (cache.keys, cache.values):
            if t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
                why = "the HIP prompt attention needs a cache of 16-byte aligned rows"
            elif t.stride(2) > MAX_ROW_STRIDE:
                why = "the HIP prompt attention needs a cache whose rows are not too far apart"
        if cache.capacity > MOST_KEYS:
            why = "the HIP prompt attention needs a block table of fewer tokens"
    return why


def prompt_attention(query, key, value, *, token_starts=None, key_starts=None, prefix=None,
                     scaling=None, softcap=None, slopes=None, window=None, workspace=None,
                     output=None, backend="auto"):
    """Attention of ``query`` (tokens, q_heads, head_dim) over ``key`` and
    ``value`` (key_tokens, kv_heads, head_dim), q_heads a multiple of kv_heads.

    Rows token_starts[b] up to token_starts[b + 1] of the query, (sequences +
    1,) int32, are sequence b's (None: all are one sequence's), key rows
    key_starts[b] up to key_starts[b + 1] its keys (None: as token_starts); the
    query rows are the last of them.  Row i sees the keys up to its own and the
    first ``prefix``[b] ((sequences,) int32) of its sequence, and of these those
    less than ``window`` tokens before it; ``scaling`` defaults to
    head_dim^-0.5, ``softcap`` and ``slopes`` are ``paged_decode``'s (the bias
    takes the distance either way).

    Returns a new tensor, or ``output``: rows that see nothing are zeros, rows of
    no sequence (all, with token_starts that decrease) zeros in a new tensor and
    left as they were in ``output``.
    An infinite or NaN key or value counts for the rows that see it alone; a row
    whose scores are -inf alone is NaN.
    ``workspace`` (a dict) keeps the buffers in which calls with few rows join
    shares of their keys; calls that share one must be ordered on one stream.
    """
    if key.ndim != 3 or key.shape != value.shape or min(key.shape[1:]) <= 0:
        raise ValueError("key and value must have the same (tokens, kv_heads, head_dim) shape")
    _check_query(query, key.shape[1], key.shape[2])
    if not query.is_floating_point():
        raise TypeError("query must be floating point")
    if any(t.dtype != query.dtype or t.device != query.device for t in (key, value)):
        raise ValueError("query, key and value must have the same device and dtype")
    sequences = 1
    if token_starts is not None:
        sequences = max(token_starts.numel() - 1, 0)
        if sequences < 1:
            raise ValueError("token_starts must have sequences + 1 entries")
        _check_int32("token_starts", token_starts, sequences + 1, query.device)
    if key_starts is None:
        if key.shape[0] != query.shape[0]:
            raise ValueError("without key_starts there are as many key rows as query rows")
    elif token_starts is None:
        raise ValueError("key_starts without token_starts")
    else:
        _check_int32("key_starts", key_starts, sequences + 1, query.device)
    if prefix is not None:
        _check_int32("prefix", prefix, sequences, query.device)
    scores = check_scores(softcap, slopes, window, query.shape[1], query.device)
    if output is not None:
        _check_output(output, query, (key, value))
    scaling = key.shape[2] ** -0.5 if scaling is None else float(scaling)
    why = _why_not_rows(query.dtype, key.shape[2])
    if pick_backend(query, backend, why is None, why) == "hip":
        return _hip.prompt_attention(query, key, value, sequences, token_starts, key_starts,
                                     prefix, scaling, scores, workspace, output)
    from .reference_paged import prompt_rows

    _check_capture(query, why or "backend='torch'")
    with torch.no_grad():
        return prompt_rows(query, key, value, token_starts, key_starts, prefix, scaling, scores,
                           output)


def paged_prompt(query, cache, *, token_starts=None, prefix=None, scaling=None, softcap=None,
                 slopes=None, window=None, workspace=None, output=None, backend="auto"):
    """Attention of the sequences' last tokens over a paged cache that holds them
    (appended before).

    Rows token_starts[b] up to token_starts[b + 1] of ``query`` (tokens,
    q_heads, head_dim) are sequence b's last tokens, ending at position
    lengths[b] - 1; without it every sequence has one.  The other arguments and
    the result as ``prompt_attention``'s.  A row that sees a token whose page is
    outside the cache is NaN, and so are those of a sequence whose length is past
    its table.  Over a ``QuantizedCache`` torch operations answer (to stay on the
    kernels, attend a prompt before it is appended, or ``paged_read`` its rows
    and ``prompt_attention`` over those).
    """
    _check_query(query, cache.heads, cache.head_dim)
    if query.dtype != cache.dtype or query.device != cache.device:
        raise ValueError("query must have the cache's dtype and device")
    _check_starts(token_starts, cache, query.shape[0])
    if prefix is not None:
        _check_int32("prefix", prefix, cache.sequences, query.device)
    scores = check_scores(softcap, slopes, window, query.shape[1], query.device)
    if output is not None:
        _check_output(output, query, ())
        if _meet_pages(output, cache):
            raise ValueError("output overlaps the cache")
    scaling = cache.head_dim ** -0.5 if scaling is None else float(scaling)
    why = _why_not_cache(cache) if query.is_cuda else None
    if pick_backend(query, backend, why is None, why) == "hip":
        return _hip.paged_prompt(query, cache, token_starts, prefix, scaling, scores, workspace,
                                 output)
    from .reference_paged import prompt_pages

    _check_capture(query, why or "backend='torch'")
    with torch.no_grad():
        return prompt_pages(query, cache, token_starts, prefix, scaling, scores, output)
