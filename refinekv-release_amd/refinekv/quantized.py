"""A paged KV cache in 4 bits.

``QuantizedCache`` stands where a ``PagedCache`` does in ``paged_append``,
``paged_read`` and ``paged_decode``, with rows and queries of a 16-bit type and
a third of the bytes: 160 a token and head at head_dim 128, where 16 bits take
512.  Every 32 dims of a row are a group with an fp16 zero (its smallest value)
and scale (a 15th of its span, rounded up to 7 significant bits) and codes of 0
to 15 that stand for zero + scale * code, so that a value is off by at most
half a scale (half of 1/15 of its group's span, 1.6 % more where the scale was
rounded up); spans below 2^-16 are held in steps of 2^-20.  A group with a value
that is not finite, or past 4096 in magnitude, stands for NaN.

The tensors hold codes and scales in the kernels' own order: ``packed`` makes a
cache of codes and scales in the plain order, ``unpacked`` gives them back.
"""

from dataclasses import dataclass, field

import torch

from . import _hip

PAGE_SIZES = (16, 32, 64, 128, 256)
GROUP_DIMS = 32
LARGEST = 4096.0
LARGEST_SCALE = 552.0  # a 15th of a span of 2 LARGEST, rounded up to 7 significant bits


def _tables(table, lengths, device):
    """The checks of a cache's block table and lengths."""
    if table.ndim != 2 or min(table.shape) <= 0 or table.dtype != torch.int32:
        raise ValueError("block_table must be int32 with a nonempty (sequences, max_blocks) shape")
    if table.shape[1] > 1 and table.stride(1) != 1:
        raise ValueError("block_table must have dense rows")
    if lengths.shape != table.shape[:1] or lengths.dtype != torch.int32:
        raise ValueError("lengths must be int32 with shape (sequences,)")
    if not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous")
    if table.device != device or lengths.device != device:
        raise ValueError("block_table and lengths must be on the cache's device")


def _check_held(codes, scales):
    """Codes of 4 bits, and on a GPU scales and zeros that the kernels' products hold
    exactly."""
    if int(codes.max()) > 15:
        raise ValueError("codes must be 0 to 15")
    if scales.device.type != "cuda":
        return
    scale, zero = scales.unbind(-1)
    odd = (scale.view(torch.int16) & 15 != 0) | (scale < 0) | (scale > LARGEST_SCALE)
    if bool((odd & ~scale.isnan()).any()):
        raise ValueError(f"scales must be NaN, or 0 to {LARGEST_SCALE:g} of 7 significant bits (their "
                         "last 4 bits 0)")
    if bool(zero.isinf().any()):
        raise ValueError("zeros must not be infinite")


def _meet(a, b):
    """Whether two contiguous tensors share memory."""
    ends = [t.data_ptr() + t.numel() * t.element_size() for t in (a, b)]
    return a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


@dataclass(frozen=True, eq=False)
class QuantizedCache:
    """Keys and values of ``sequences`` sequences in pages, in 4 bits.

    ``key_codes``/``value_codes``: (pages, kv_heads, page_size, head_dim / 2)
    uint8, ``key_scales``/``value_scales``: (pages, kv_heads, page_size,
    head_dim / 32, 2) float16, all contiguous, apart from each other and (on a
    GPU) 16-byte aligned.  ``block_table`` and ``lengths`` as a ``PagedCache``'s.
    ``dtype`` is the rows' and queries', bfloat16 or float16.  The tensors'
    contents may change; their sizes and strides are read once.
    """

    key_codes: torch.Tensor
    value_codes: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    block_table: torch.Tensor
    lengths: torch.Tensor
    dtype: torch.dtype = torch.bfloat16
    pages: int = field(init=False)
    heads: int = field(init=False)
    page_size: int = field(init=False)
    head_dim: int = field(init=False)
    sequences: int = field(init=False)
    max_blocks: int = field(init=False)
    device: torch.device = field(init=False)

    def __post_init__(self):
        codes, scales = (self.key_codes, self.value_codes), (self.key_scales, self.value_scales)
        shape, device = self.key_codes.shape, self.key_codes.device
        if len(shape) != 4 or min(shape) <= 0 or self.value_codes.shape != shape:
            raise ValueError("codes must have the same nonempty (pages, kv_heads, page_size, "
                             "head_dim / 2) shape")
        dim = 2 * shape[3]
        if dim not in _hip.SUPPORTED_DIMS:
            raise ValueError("a cache in 4 bits needs head_dim in 32..256 (multiple of 32)")
        if shape[2] not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if any(t.shape != (*shape[:3], dim // GROUP_DIMS, 2) for t in scales):
            raise ValueError("scales must have shape (pages, kv_heads, page_size, head_dim / 32, "
                             "2)")
        if any(t.dtype != torch.uint8 for t in codes):
            raise TypeError("codes must be uint8")
        if any(t.dtype != torch.float16 for t in scales):
            raise TypeError("scales must be float16")
        if self.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("a cache in 4 bits takes bfloat16 or float16 rows")
        parts = (*codes, *scales)
        if any(t.device != device for t in parts):
            raise ValueError("codes and scales must be on the same device")
        if not all(t.is_contiguous() for t in parts):
            raise ValueError("codes and scales must be contiguous")
        if any(_meet(a, b) for i, a in enumerate(parts) for b in parts[i + 1:]):
            raise ValueError("codes and scales must not share memory")
        if device.type == "cuda" and any(t.data_ptr() % 16 for t in parts):
            raise ValueError("codes and scales must be 16-byte aligned")
        _tables(self.block_table, self.lengths, device)
        sizes = dict(pages=shape[0], heads=shape[1], page_size=shape[2], head_dim=dim,
                     sequences=self.block_table.shape[0], max_blocks=self.block_table.shape[1],
                     device=device)
        for name, value in sizes.items():
            object.__setattr__(self, name, value)

    def __getstate__(self):
        # (copies look up anew what the calls have noted about these tensors)
        return {k: v for k, v in self.__dict__.items() if not k.startswith("_hip")}

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, sequences, max_blocks, *,
              dtype=torch.bfloat16, device=None):
        """A new cache of zeros with no pages assigned (block_table -1)."""
        if head_dim not in _hip.SUPPORTED_DIMS:
            raise ValueError("a cache in 4 bits needs head_dim in 32..256 (multiple of 32)")
        shape = (pages, kv_heads, page_size)
        codes = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device)
                 for _ in range(2)]
        scales = [torch.zeros(*shape, head_dim // GROUP_DIMS, 2, dtype=torch.float16,
                              device=device) for _ in range(2)]
        return cls(*codes, *scales,
                   torch.full((sequences, max_blocks), -1, dtype=torch.int32, device=device),
                   torch.zeros(sequences, dtype=torch.int32, device=device), dtype)

    @classmethod
    def packed(cls, key_codes, value_codes, key_scales, value_scales, block_table, lengths, *,
               dtype=torch.bfloat16):
        """A cache of codes (pages, kv_heads, page_size, head_dim) uint8, one a
        byte, and (scale, zero) pairs (pages, kv_heads, page_size,
        head_dim / 32, 2) float16; both are copied.

        On a GPU scales must have 7 significant bits (their last 4 bits 0) and
        lie in 0..552, or be NaN, and zeros not be infinite, in every page: the
        kernels' products hold no others (the torch operations on a CPU take
        them all; a cache that is moved to a GPU is not looked at again)."""
        for codes, scales in ((key_codes, key_scales), (value_codes, value_scales)):
            if codes.ndim != 4 or codes.dtype != torch.uint8 or codes.shape[3] % GROUP_DIMS or (
                    codes.shape[2] % 16):
                raise ValueError("codes must be uint8 with shape (pages, kv_heads, page_size, "
                                 "head_dim)")
            if scales.dtype != torch.float16 or scales.shape != (
                    *codes.shape[:3], codes.shape[3] // GROUP_DIMS, 2):
                raise ValueError("scales must be float16 with shape (pages, kv_heads, page_size, "
                                 "head_dim / 32, 2)")
            if codes.numel():
                _check_held(codes, scales)
        return cls(pack_keys(key_codes), pack_values(value_codes), key_scales.clone(
            memory_format=torch.contiguous_format), pack_scales(value_scales), block_table,
            lengths, dtype)

    def unpacked(self):
        """(key_codes, value_codes, key_scales, value_scales) as ``packed``
        takes them."""
        return (unpack_keys(self.key_codes), unpack_values(self.value_codes),
                self.key_scales.clone(), unpack_scales(self.value_scales))

    @property
    def capacity(self):
        """Tokens a sequence's row of the table can address."""
        return self.max_blocks * self.page_size


# ---------------------------------------------------------------------------
# The kernels' order
# ---------------------------------------------------------------------------

def _bytes(nibbles):
    """(.., 2) codes, low first, as bytes."""
    return nibbles[..., 0] | (nibbles[..., 1] << 4)


def _nibbles(data):
    return torch.stack((data & 15, data >> 4), -1)


def pack_keys(codes):
    """A row's dwords lie by lane row (of 8 dims) and group; the even dims of a
    dword in its low half, the odd ones in its high half."""
    x = codes.unflatten(-1, (-1, 4, 4, 2))  # group, lane row, pair, dim of the pair
    x = x.movedim((-4, -3, -2, -1), (-3, -4, -1, -2)).flatten(-4).unflatten(-1, (-1, 2))
    return _bytes(x).contiguous()


def unpack_keys(data):
    x = _nibbles(data).flatten(-2).unflatten(-1, (4, -1, 2, 4))  # lane row, group, dim, pair
    return x.movedim((-4, -3, -2, -1), (-3, -4, -1, -2)).flatten(-4).contiguous()


def _pieces(dim):
    """(first dim, dims of a column) of a row's pieces: 128 dims each, then 64,
    then 32."""
    whole = dim // 128 * 128
    found = [(d, 8) for d in range(0, whole, 128)]
    if dim - whole >= 64:
        found.append((whole, 4))
        whole += 64
    if dim - whole >= 32:
        found.append((whole, 2))
    return found


def pack_values(codes):
    """Blocks of 4 tokens: by piece and column, entries (token pair, dim) of
    two tokens' codes, four a dword."""
    blocks = codes.unflatten(-2, (-1, 4))
    parts = []
    for first, dims in _pieces(codes.shape[-1]):
        x = blocks[..., first:first + 16 * dims].unflatten(-1, (16, dims)).unflatten(-3, (2, 2))
        # pair, token, column, dim -> column, (pair, dim), token
        x = x.movedim((-4, -3, -2, -1), (-3, -1, -4, -2)).flatten(-3, -2)
        x = x.unflatten(-2, (-1, 4)).transpose(-1, -2)  # dword, token, entry
        parts.append(_bytes(x.flatten(-4).unflatten(-1, (-1, 2))))
    shape = (*codes.shape[:-1], codes.shape[-1] // 2)
    return torch.cat(parts, -1).reshape(shape)


def unpack_values(data):
    dim = 2 * data.shape[-1]
    blocks = data.unflatten(-2, (-1, 4)).flatten(-2)
    parts, at = [], 0
    for first, dims in _pieces(dim):
        x = _nibbles(blocks[..., at:at + 32 * dims]).flatten(-2)
        at += 32 * dims
        x = x.unflatten(-1, (16, -1, 2, 4)).transpose(-1, -2).flatten(-3, -2)  # column, entry, token
        x = x.unflatten(-2, (2, dims)).movedim((-4, -3, -2, -1), (-2, -4, -1, -3))
        parts.append(x.flatten(-2).flatten(-3, -2))  # 4 tokens, the piece's dims
    return torch.cat(parts, -1).flatten(-3, -2)


def pack_scales(scales):
    """Of values: a group's scales of 4 tokens, then their zeros."""
    return scales.unflatten(-3, (-1, 4)).movedim(-3, -1).contiguous().view(scales.shape)


def unpack_scales(data):
    shape = data.shape
    blocks = data.unflatten(-3, (-1, 4)).flatten(-3).unflatten(-1, (shape[-2], 2, 4))
    return blocks.movedim(-1, -3).reshape(shape)


# ---------------------------------------------------------------------------
# The format, in torch operations
# ---------------------------------------------------------------------------

def quantize(rows):
    """(codes, (scale, zero) pairs) of (.., dim) rows, in the plain order."""
    x = rows.float().unflatten(-1, (-1, GROUP_DIMS))
    low, high = x.amin(-1), x.amax(-1)
    near = ((high - low) / 15.0).half()
    scale = ((near.view(torch.int16) + 15) & -16).view(torch.float16)
    held = torch.maximum(low.abs(), high.abs()) <= LARGEST  # (false for NaN)
    pairs = torch.where(held[..., None], torch.stack((scale, low.half()), -1), torch.nan)
    step, base = pairs.float()[..., None].unbind(-2)
    codes = ((x - base) / step).round().clamp(0.0, 15.0)
    codes = torch.where(held[..., None] & (step > 0), codes, 0.0).to(torch.uint8)
    return codes.flatten(-2), pairs


def dequantize(codes, scales):
    """What codes and scales in the plain order stand for, in 32 bits."""
    scale, zero = scales.float()[..., None].unbind(-2)
    return (codes.float().unflatten(-1, (-1, GROUP_DIMS)) * scale + zero).flatten(-2)
