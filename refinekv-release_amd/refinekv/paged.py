"""A KV cache in pages shared by many sequences, and the attention over it.

The reference's caches hold one sequence, contiguous; a server that decodes
many at once keeps their tokens in pages of one allocation.  ``PagedCache``
describes such a cache (the tensors are the caller's, and so is the
allocation of pages), ``paged_append`` writes new keys and values to it,
turned to their positions on the way, and ``paged_decode`` attends one new
token per sequence over its visible tokens.  A decode step::

    cache.lengths.add_(1)                 # the new token counts as visible
    query = paged_append(key, value, cache, query=query, rotary=rotary)
    output = paged_decode(query, cache, workspace=workspace)

The kernels read lengths and block table on the device, so one captured HIP
graph serves every step of a batch.  ROCm tensors use the gfx950 kernels,
others (and the types and shapes the kernels do not take) torch operations,
which read lengths on the host: those calls cannot be captured and say so.
Inference only, as the whole package: the results carry no gradient.
"""

from dataclasses import dataclass, field

import torch

from . import _hip
from .rotary import DTYPES, check_out, overlaps_itself, pick_backend, rows_overlap

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_ROW_STRIDE = 1 << 25  # elements between a page's rows, at most


@dataclass(frozen=True, eq=False)
class PagedCache:
    """Keys and values of ``sequences`` sequences in pages.

    ``keys``/``values``: (pages, kv_heads, page_size, head_dim), head_dim
    dense, the other strides free (a cache kept as (pages, page_size,
    kv_heads, head_dim) is passed as its transposed view).  ``block_table``:
    (sequences, max_blocks) int32, the page of each page_size tokens; entries
    past a sequence's length are not read.  ``lengths``: (sequences,) int32,
    the visible tokens, those being appended included; 0 marks an idle place.
    The tensors' contents may change; their sizes, strides and alignment are
    read once.
    """

    keys: torch.Tensor
    values: torch.Tensor
    block_table: torch.Tensor
    lengths: torch.Tensor
    pages: int = field(init=False)
    heads: int = field(init=False)
    page_size: int = field(init=False)
    head_dim: int = field(init=False)
    sequences: int = field(init=False)
    max_blocks: int = field(init=False)
    dtype: torch.dtype = field(init=False)
    device: torch.device = field(init=False)

    def __post_init__(self):
        keys, values, table, lengths = self.keys, self.values, self.block_table, self.lengths
        if keys.ndim != 4 or keys.shape != values.shape or min(keys.shape) <= 0:
            raise ValueError("keys and values must have the same nonempty (pages, kv_heads, "
                             "page_size, head_dim) shape")
        if keys.dtype != values.dtype or keys.device != values.device:
            raise ValueError("keys and values must have the same device and dtype")
        if not keys.is_floating_point():
            raise TypeError("keys and values must be floating point")
        if keys.shape[2] not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if keys.shape[3] > 1 and (keys.stride(3) != 1 or values.stride(3) != 1):
            raise ValueError("keys and values must have a dense head_dim")
        if overlaps_itself(keys) or overlaps_itself(values):
            raise ValueError("keys and values must not overlap themselves")
        if table.ndim != 2 or min(table.shape) <= 0 or table.dtype != torch.int32:
            raise ValueError("block_table must be int32 with a nonempty (sequences, max_blocks) "
                             "shape")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("block_table must have dense rows")
        if lengths.shape != table.shape[:1] or lengths.dtype != torch.int32:
            raise ValueError("lengths must be int32 with shape (sequences,)")
        if not lengths.is_contiguous():
            raise ValueError("lengths must be contiguous")
        if table.device != keys.device or lengths.device != keys.device:
            raise ValueError("block_table and lengths must be on the cache's device")
        sizes = dict(zip(("pages", "heads", "page_size", "head_dim"), keys.shape),
                     sequences=table.shape[0], max_blocks=table.shape[1], dtype=keys.dtype,
                     device=keys.device)
        for name, value in sizes.items():
            object.__setattr__(self, name, value)

    def __getstate__(self):
        # (copies look up anew what the calls have noted about these tensors)
        return {k: v for k, v in self.__dict__.items() if not k.startswith("_hip")}

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, sequences, max_blocks, *,
              dtype=torch.bfloat16, device=None):
        """A new cache of zeros with no pages assigned (block_table -1)."""
        shape = (pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device),
                   torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((sequences, max_blocks), -1, dtype=torch.int32, device=device),
                   torch.zeros(sequences, dtype=torch.int32, device=device))

    @property
    def capacity(self):
        """Tokens a sequence's row of the table can address."""
        return self.max_blocks * self.page_size


def _check_rows(name, rows, cache, tokens, heads=None):
    shape = rows.shape
    if (len(shape) != 3 or shape[0] != tokens or shape[2] != cache.head_dim
            or (shape[1] <= 0 if heads is None else shape[1] != heads)):
        raise ValueError(f"{name} must have shape (tokens, heads, head_dim) with the key's "
                         "tokens and the cache's head_dim and, keys and values, heads")
    if rows.dtype != cache.dtype or rows.device != cache.device:
        raise ValueError(f"{name} must have the cache's dtype and device")


def _check_capture(rows, why):
    """The torch operations ask the device for values, which a capture does not
    allow."""
    if rows.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"this call cannot be captured in a graph: {why}")


def _keys_meet_values(cache):
    """Whether the cache's keys and values may share memory: the C entry's own
    rule, for the torch operations."""
    size = cache.keys.element_size()
    axes = sorted(((s * size, t * size, n) for s, t, n in
                   zip(cache.keys.stride(), cache.values.stride(), cache.keys.shape) if n > 1),
                  reverse=True)

    def meet(level, apart):
        keys, values = (size + sum((a[2] - 1) * a[i] for a in axes[level:]) for i in (0, 1))
        if apart >= keys or -apart >= values:
            return False
        if level == len(axes):
            return True
        stride, other, count = axes[level]
        if stride != other:
            return True
        keys, values = keys - (count - 1) * stride, values - (count - 1) * stride
        steps = range(max(-((values - 1 + apart) // stride), 1 - count),
                      min((keys - 1 - apart) // stride, count - 1) + 1)
        return len(steps) > 3 or any(meet(level + 1, apart + d * stride) for d in steps)

    return meet(0, cache.values.data_ptr() - cache.keys.data_ptr())


def _meet_pages(rows, cache):
    """Whether (tokens, heads, head_dim) rows may lie among the cache's pages,
    by the C entries' rule: their spans meet."""
    def span(t):
        first, size = t.data_ptr(), t.element_size()
        return first, first + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))

    if rows.numel() == 0:
        return False
    first, end = span(rows)
    return any(first < e and f < end for f, e in map(span, (cache.keys, cache.values)))


def paged_append(key, value, cache, *, query=None, rotary=None, token_starts=None,
                 query_out=None, backend="auto"):
    """Write new (tokens, kv_heads, head_dim) keys and values to their
    sequences' pages, and return the turned queries (None without a query).

    With ``token_starts`` (sequences + 1,) int32, rows token_starts[b] up to
    token_starts[b + 1] are sequence b's last tokens, ending at position
    lengths[b] - 1; without it every sequence has one.  With ``rotary`` keys
    and ``query`` (tokens, q_heads, head_dim) are turned to those positions;
    ``query_out`` takes the turned queries (it may be the query itself, but not
    lie in the cache).

    Rows of no sequence (behind the last one) or without a position (an idle
    place: length 0) are not stored, and their queries are returned unturned.
    A row whose page is outside the cache, or past the block table, is not
    stored.  No two rows of a call may fall on the same place: a page written
    here belongs to one sequence, and a cache whose keys and values share
    memory is refused.  Rows that are views of the cache's pages are copied
    first: the call stores what they hold before it.

    (A prompt's own attention needs its turned keys as well: turn both with
    rotate_heads, then append without ``rotary``.)
    """
    tokens, device = key.shape[0] if key.ndim else 0, cache.device
    _check_rows("key", key, cache, tokens, cache.heads)
    _check_rows("value", value, cache, tokens, cache.heads)
    if token_starts is not None:
        if (token_starts.shape != (cache.sequences + 1,) or token_starts.dtype != torch.int32
                or token_starts.device != device or not token_starts.is_contiguous()):
            raise ValueError("token_starts must be contiguous int32 with shape (sequences + 1,) "
                             "on the cache's device")
    elif tokens != cache.sequences:
        raise ValueError("without token_starts there is one token per sequence")
    if rotary is not None and (rotary.config.head_dim != cache.head_dim
                               or rotary.device != device):
        raise ValueError("rotary must have the cache's head_dim and device")
    if query is not None:
        if rotary is None:
            raise ValueError("a query is only taken to be turned: pass rotary")
        _check_rows("query", query, cache, tokens)
        if query_out is not None:
            check_out("query_out", query_out, query, (key, value))
    elif query_out is not None:
        raise ValueError("query_out without a query")
    why = None if key.dtype in DTYPES else "the HIP append needs a bf16, fp16 or fp32 cache"
    if pick_backend(key, backend, why is None, why) == "hip":
        return _hip.paged_append(key, value, cache, query, rotary, token_starts, query_out)
    from .reference_paged import append

    _check_capture(key, why or "backend='torch'")

    if _keys_meet_values(cache):
        raise ValueError("the cache's keys and values share memory")
    if query_out is not None and _meet_pages(query_out, cache):
        raise ValueError("query_out overlaps the cache")
    with torch.no_grad():
        turned = append(cache, key, value, query, rotary, token_starts)
        return turned if query_out is None else query_out.copy_(turned)


def _decode_support(cache, group):
    """None, or why the HIP kernel does not take the cache with this group;
    looked up once (a frozen cache's tensors keep their layout)."""
    known = cache.__dict__.setdefault("_hip_support", {})
    if group not in known:
        known[group] = _why_not(cache, group)
    return known[group]


def _why_not(cache, group):
    dim = cache.head_dim
    if cache.dtype not in (torch.bfloat16, torch.float16):
        return "the HIP paged decode needs a bf16 or fp16 cache"
    if dim not in _hip.SUPPORTED_DIMS or group > _hip.MAX_GROUP:
        return "the HIP paged decode needs head_dim in 32..256 (multiple of 32) and group <= 16"
    for t in (cache.keys, cache.values):
        if t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:3], t.shape) if n > 1):
            return "the HIP paged decode needs a cache of 16-byte aligned rows"
        if not dim <= t.stride(2) <= MAX_ROW_STRIDE:
            return "the HIP paged decode needs rows apart from each other, and not too far"
    if cache.sequences * cache.heads * (cache.capacity // 32 + 1) >= 2 ** 31:
        return "the HIP paged decode needs a block table of fewer tokens"
    return None


def paged_decode(query, cache, *, scaling=None, workspace=None, output=None, backend="auto"):
    """Attention of one new token per sequence over its visible tokens.

    ``query`` (sequences, q_heads, head_dim), q_heads a multiple of the
    cache's heads (head h's rows are its group h); ``scaling`` defaults to
    head_dim^-0.5.  Returns a new tensor of the query's shape, or ``output``
    (apart from the query and the cache).
    ``workspace`` (a dict) keeps the partial results' buffer from call to
    call; calls that share one must be ordered on one stream.

    A sequence of length 0 gives zeros; one with a page outside the cache
    among its visible ones, or a length past its table, gives NaN.
    """
    _check_rows("query", query, cache, cache.sequences)
    group = query.shape[1] // cache.heads
    if query.shape[1] != group * cache.heads:
        raise ValueError("query heads must be a multiple of the cache's heads")
    if output is not None:
        if (output.shape != query.shape or output.dtype != query.dtype
                or output.device != query.device or not output.is_contiguous()):
            raise ValueError("output must be contiguous with the query's shape, dtype and device")
        if rows_overlap(output, query):
            raise ValueError("output must not overlap the query")
    scaling = cache.head_dim ** -0.5 if scaling is None else float(scaling)
    why = _decode_support(cache, group) if query.is_cuda else None
    hip = pick_backend(query, backend, why is None, why) == "hip"
    if hip and (output is None or output.data_ptr() % 16 == 0):
        return _hip.paged_decode(query, cache, scaling, workspace, output)
    if not hip:
        _check_capture(query, why or "backend='torch'")
    from .reference_paged import decode

    if output is not None and _meet_pages(output, cache):
        raise ValueError("output overlaps the cache")
    if hip:  # (the kernel stores whole vectors)
        return output.copy_(_hip.paged_decode(query, cache, scaling, workspace))
    with torch.no_grad():
        out = decode(query, cache, scaling)
        return out if output is None else output.copy_(out)
