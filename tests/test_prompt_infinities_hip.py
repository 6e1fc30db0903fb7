"""Infinite and NaN keys and values far below a row's largest score (GPU).

They count for every row that sees them, however little they weigh, and for no
other; the same in 64 bits says which rows those are (weights of e^-700 are not
0 there)."""

import math

import pytest
import torch

from prompt_math import assert_rows, prompt64
from refinekv import prompt_attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    from refinekv import _hip

    _hip.lib()  # the HIP library must load: no fallback
    return _hip


def rows(n, heads, dim, dtype, gen):
    return torch.randn(n, heads, dim, generator=gen).to(dtype)


def early(value, at):
    """Values that are not finite in the first rows from `at` on, dims apart."""
    value[at, :, 3], value[at + 1, :, 5], value[at + 2, :, 7] = math.inf, -math.inf, math.nan
    value[at + 3, :, 9], value[at + 4, :, 9] = math.inf, -math.inf


def check(query, key, value, starts, key_starts, **options):
    on_gpu = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in options.items()}
    ends = {} if key_starts is starts else dict(key_starts=key_starts.to(DEV))
    got = prompt_attention(*(t.to(DEV) for t in (query, key, value)),
                           token_starts=starts.to(DEV), backend="hip", **ends, **on_gpu)
    want, room = prompt64(query, key, value, starts, key_starts, **options)
    # (what the bounds are for: each kind is there, and rows without any)
    assert bool((want == math.inf).any()) and bool((want == -math.inf).any())
    assert bool(want.isnan().any()) and bool(want.isfinite().any())
    assert_rows(got, want, room, str([k for k in options]))


@pytest.mark.parametrize("dim,dtype", [(32, F16), (64, BF16), (96, BF16), (128, F16), (128, BF16),
                                       (256, BF16)])
def test_values_far_behind(dim, dtype):
    """Up to 250 tokens back with slopes of up to 1, and with scores that rise by
    1 a token: weights down to e^-250."""
    gen = torch.Generator().manual_seed(dim)
    starts = torch.tensor([0, 250, 287], dtype=torch.int32)
    query, key, value = (rows(287, n, dim, dtype, gen) for n in (4, 2, 2))
    early(value, 0)
    early(value, 261)
    check(query, key, value, starts, starts, slopes=torch.tensor([1.0, 0.7, 0.5, 0.3]))
    check(query, key, value, starts, starts, slopes=torch.tensor([1.0, 0.7, 0.5, 0.3]),
          prefix=torch.tensor([100, 0], dtype=torch.int32), window=200)
    query[..., :2], key[..., :2] = 1.0, 0.0
    key[:, :, 0] = (torch.arange(287) % 250)[:, None]
    check(query, key, value, starts, starts, scaling=1.0)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (160, BF16)])
def test_values_far_behind_in_shares(dim, dtype):
    """Few rows, whose keys several workgroups share: a part that weighs e^-600
    beside another, infinite or NaN."""
    gen = torch.Generator().manual_seed(dim)
    starts = torch.tensor([0, 40, 45], dtype=torch.int32)
    key_starts = torch.tensor([0, 3000, 4000], dtype=torch.int32)
    query = rows(45, 4, dim, dtype, gen)
    key, value = (rows(4000, 2, dim, dtype, gen) for _ in range(2))
    early(value, 0)
    early(value, 2988)  # (and the last rows of the first sequence alone)
    slopes = torch.tensor([0.2, 0.15, 0.1, 0.05])
    check(query, key, value, starts, key_starts, slopes=slopes)
    check(query, key, value, starts, key_starts, slopes=-slopes)
    check(query, key, value, starts, key_starts, slopes=slopes, window=2975)
