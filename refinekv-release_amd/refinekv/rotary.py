"""Rotary positions of query and key heads.

The reference leaves them to the model (its hook calls the model's own
function on the anchor queries, src/refinekv/integrations/transformers.py:485-508);
serving over a paged cache needs them beside the cache write.  ``RotaryConfig``
describes the rotation, ``Rotary`` holds its rates on a device and
``rotate_heads`` turns rows of heads; ``paged_append`` (paged.py) turns them on
the way into the cache.  ROCm tensors use the gfx950 kernel, others torch
operations; both reduce the angles in 64 bits, multiply in 32 and round once.
Inference only, as the whole package: the results carry no gradient
(``inverse=True`` is the transposed rotation).
"""

from dataclasses import dataclass
import math

import torch

from . import _hip
from .config import BACKENDS, KERNEL_BACKENDS

SCALINGS = ("none", "linear", "ntk", "llama3", "yarn")
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
POSITION_DTYPES = (torch.int64, torch.int32)


@dataclass(frozen=True)
class RotaryConfig:
    """How a head's pairs turn with the position.

    ``rotary_dim`` (even, default the whole head) leading dims turn, the rest
    pass; pair i turns by position * base^(-2 i / rotary_dim) radians.  Pairs
    are dims (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if ``interleaved``.
    ``scaling`` stretches the rates for contexts longer than
    ``original_length``: ``linear`` divides them by ``factor``; ``ntk`` raises
    the base by factor^(rotary_dim / (rotary_dim - 2)); ``llama3`` divides
    those whose wavelength passes original_length / low_freq_factor, keeps
    those under original_length / high_freq_factor and blends between;
    ``yarn`` blends between the pairs that turn ``beta_fast`` and ``beta_slow``
    times within original_length and multiplies the turned dims by
    ``attention_factor`` (default 0.1 ln(factor) + 1).
    """

    head_dim: int
    rotary_dim: int | None = None
    base: float = 10000.0
    interleaved: bool = False
    scaling: str = "none"
    factor: float = 1.0
    original_length: int = 8192
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self):
        for name in ("head_dim", "original_length"):
            value = getattr(self, name)
            if not isinstance(value, int) or isinstance(value, bool) or value <= 0:
                raise ValueError(f"{name} must be a positive integer")
        if self.rotary_dim is None:
            object.__setattr__(self, "rotary_dim", self.head_dim)
        dim = self.rotary_dim
        if (not isinstance(dim, int) or isinstance(dim, bool) or dim <= 0 or dim % 2
                or dim > self.head_dim):
            raise ValueError("rotary_dim must be even and in 2..head_dim")
        if not math.isfinite(self.base) or self.base <= 1:
            raise ValueError("base must be finite and above 1")
        if self.scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}")
        if not math.isfinite(self.factor) or self.factor < 1:
            raise ValueError("factor must be finite and at least 1")
        if self.scaling == "ntk" and dim == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        if not 0 < self.low_freq_factor < self.high_freq_factor < math.inf:
            raise ValueError("low_freq_factor must be positive and below high_freq_factor")
        if not 0 < self.beta_slow < self.beta_fast < math.inf:
            raise ValueError("beta_slow must be positive and below beta_fast")
        if self.attention_factor is not None and not (math.isfinite(self.attention_factor)
                                                      and self.attention_factor > 0):
            raise ValueError("attention_factor must be finite and positive")

    def rates(self):
        """Radians per position of each pair, as Python floats."""
        dim, factor, length = self.rotary_dim, self.factor, self.original_length
        base = self.base
        if self.scaling == "ntk":
            base *= factor ** (dim / (dim - 2))
        rates = [base ** (-2 * i / dim) for i in range(dim // 2)]
        if self.scaling == "linear":
            return [rate / factor for rate in rates]
        if self.scaling == "llama3":
            def keep(rate):  # the share of the unscaled rate
                turns = length * rate / (2 * math.pi)
                share = ((turns - self.low_freq_factor)
                         / (self.high_freq_factor - self.low_freq_factor))
                return min(max(share, 0.0), 1.0)
        elif self.scaling == "yarn":
            def pair(turns):  # the pair that turns so often within length
                return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

            low = max(math.floor(pair(self.beta_fast)), 0)
            high = min(math.ceil(pair(self.beta_slow)), dim - 1)
            span = max(high - low, 0.001)
            index = iter(range(len(rates)))

            def keep(rate):
                return 1 - min(max((next(index) - low) / span, 0.0), 1.0)
        else:
            return rates
        shares = [keep(rate) for rate in rates]
        return [rate * (share + (1 - share) / factor) for rate, share in zip(rates, shares)]

    @property
    def output_scale(self):
        """The factor on the turned dims (yarn's attention factor)."""
        if self.attention_factor is not None:
            return float(self.attention_factor)
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" else 1.0


class Rotary:
    """A RotaryConfig's rates on a device: ``turns`` (rotary_dim / 2,) float64,
    whole turns per position, and ``scale``.  ``rates`` replaces the config's
    radians per position (a model's own inverse frequencies)."""

    def __init__(self, config, device=None, rates=None):
        if not isinstance(config, RotaryConfig):
            raise TypeError("Rotary needs a RotaryConfig")
        self.config = config
        rates = torch.as_tensor(config.rates() if rates is None else rates, dtype=torch.float64)
        if rates.shape != (config.rotary_dim // 2,):
            raise ValueError("rates must have rotary_dim / 2 entries")
        self.turns = (rates / (2 * math.pi)).to(device if device is not None else rates.device)
        self.scale = config.output_scale

    @property
    def device(self):
        return self.turns.device


def pick_backend(tensor, backend, supported, why):
    """"hip" or "torch" for a call on ``tensor``: the kernels where they run
    (``supported``; an explicit request otherwise raises ``why``), never a
    silent fallback for a missing library on a GPU."""
    if backend not in BACKENDS:
        raise ValueError("backend must be 'auto', 'torch', 'hip', or 'triton'")
    if backend == "torch":
        return "torch"
    explicit = backend in KERNEL_BACKENDS
    if not _hip.is_rocm_device(tensor):
        if explicit:
            raise RuntimeError("the HIP backend requires a ROCm GPU tensor")
        return "torch"
    if not supported:
        if explicit:
            raise TypeError(why)
        return "torch"
    _hip.lib()
    return "hip"


def _extent(sizes, strides):
    return sum((n - 1) * s for n, s in zip(sizes, strides)) + 1


def rows_overlap(a, b):
    """Whether the memory of two (rows, heads, dim) views may overlap: their
    spans meet, and they are not separate columns of one row-major matrix."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size = a.element_size()
    ea, eb = (_extent(t.shape, t.stride()) * t.element_size() for t in (a, b))
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + ea <= pb or pb + eb <= pa:
        return False
    pitch = a.stride(0) * size
    if a.stride(0) != b.stride(0) or size != b.element_size() or pitch == 0:
        return True
    ra, rb = (_extent(t.shape[1:], t.stride()[1:]) * size for t in (a, b))
    gap = (pb - pa) % pitch
    return not (gap >= ra and gap + rb <= pitch)


def overlaps_itself(t):
    """Whether two elements of a strided view may share memory."""
    inner = 1
    for stride, count in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < inner:
            return True
        inner += stride * (count - 1)
    return False


def check_out(name, out, like, others=()):
    """``out`` can take rows like ``like``'s, in place of them or apart from
    every tensor in ``others``."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must have its input's shape, dtype and device")
    if overlaps_itself(out):
        raise ValueError(f"{name} must not overlap itself")
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError(f"{name} must have a dense head_dim")
    same = out.data_ptr() == like.data_ptr() and out.stride() == like.stride()
    for other in others if same else (like, *others):
        if rows_overlap(out, other):
            raise ValueError(f"{name} overlaps an input or output of the call")


def rotate_heads(query, key, positions, rotary, *, query_out=None, key_out=None, inverse=False,
                 backend="auto"):
    """Turn (tokens, heads, head_dim) query and key rows to their positions.

    ``positions`` (tokens,) int32 or int64, of less than 2^49 turns; ``key``
    may be None.  Returns
    (query, key), new tensors unless ``query_out`` / ``key_out`` are given,
    which may be the inputs themselves.  ``inverse`` turns by the opposite
    angles (the factor of a yarn rotation multiplies either way).
    """
    config, shape, dtype, device = rotary.config, query.shape, query.dtype, query.device
    if len(shape) != 3 or shape[1] <= 0 or shape[2] != config.head_dim:
        raise ValueError("query must have shape (tokens, heads, head_dim) of the rotary's head_dim")
    if not dtype.is_floating_point:
        raise TypeError("query must be floating point")
    if key is not None:
        kv = key.shape
        if len(kv) != 3 or kv[0] != shape[0] or kv[1] <= 0 or kv[2] != shape[2]:
            raise ValueError("key must have shape (tokens, heads, head_dim) with the query's "
                             "tokens and head_dim")
        if key.dtype != dtype or key.device != device:
            raise ValueError("query and key must have the same device and dtype")
    elif key_out is not None:
        raise ValueError("key_out without a key")
    if positions.shape != shape[:1] or positions.dtype not in POSITION_DTYPES:
        raise ValueError("positions must be int32 or int64 with shape (tokens,)")
    if positions.device != device or rotary.turns.device != device:
        raise ValueError("positions and rotary must be on the query device")
    if query_out is not None:
        check_out("query_out", query_out, query, [t for t in (key, key_out) if t is not None])
    if key_out is not None:
        check_out("key_out", key_out, key, [query])
    if pick_backend(query, backend, dtype in DTYPES,
                    "the HIP rotation needs bf16, fp16 or fp32 rows") == "hip":
        return _hip.rotary(query, key, positions, rotary, query_out, key_out, inverse)
    from .reference_paged import rotate

    rows = []
    with torch.no_grad():
        for x, out in ((query, query_out), (key, key_out)):
            if x is not None:
                y = rotate(x, positions, rotary, inverse)
                x = y if out is None else out.copy_(y)
            rows.append(x)
    return tuple(rows)
