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


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (256, BF16)])
def test_scores_of_minus_infinity(dim, dtype):
    """Rows whose seen keys all score -inf are NaN, as a softmax's; such keys
    weigh nothing beside others; rows that see no key are zeros."""
    gen = torch.Generator().manual_seed(dim)
    query, key, value = (rows(150, n, dim, dtype, gen) for n in (4, 2, 2))
    query[..., 0] = 1.0
    key[:3, :, 0] = -math.inf
    key[149, :, 0] = -math.inf
    value[149, :, 5] = math.inf  # (a NaN row has no infinities)
    on_gpu = [t.to(DEV) for t in (query, key, value)]
    starts = torch.tensor([0, 149], dtype=torch.int32)
    at = starts.to(DEV)
    got = prompt_attention(*on_gpu, token_starts=at, backend="hip")
    assert bool(got[:3].isnan().all())
    want, room = prompt64(query, key, value, [3, 149], [3, 149])
    assert_rows(got[3:149], want[3:149], room[3:149])
    got = prompt_attention(*on_gpu, window=1, backend="hip")  # each row its own token
    alone = torch.tensor([0, 1, 2, 149], device=DEV)
    assert bool(got[alone].isnan().all()) and bool(got[3:149].isfinite().all())
    # 5 rows over 3000 keys and 700 over 600, which are shared out
    counts, lengths = [5, 700], [3000, 600]
    starts, ends = (torch.tensor([0] + n).cumsum(0).int() for n in (counts, lengths))
    query = rows(705, 1, dim, dtype, gen)
    key, value = (rows(3600, 1, dim, dtype, gen) for _ in range(2))
    query[..., 0] = 1.0
    key[:3000, 0, 0] = -math.inf
    value[1000, 0, 7] = math.inf
    got = prompt_attention(*(t.to(DEV) for t in (query, key, value)), token_starts=starts.to(DEV),
                           key_starts=ends.to(DEV), backend="hip")
    assert bool(got[:5].isnan().all())
    want, room = prompt64(query, key, value, [5, 705], [3000, 3600])
    assert_rows(got[5:], want[5:], room[5:])
    assert not bool(got[5:105].any())
