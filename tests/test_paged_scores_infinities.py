"""Infinite values under capped, biased and windowed scores of the paged decode:
as without them an infinity makes its dim infinite, and NaN where its weight is 0
or one of the other sign is there; what a window hides does not count."""

import math

import pytest
import torch

from paged_math import pages_for
from refinekv import PagedCache, paged_decode


def check(device, backend):
    gen = torch.Generator().manual_seed(3)
    n, dim = 700, 64
    keys, values, table = pages_for([n], 16, 2, dim, torch.bfloat16, gen)

    def put(token, at, value):
        values[int(table[0, token // 16]), :, token % 16, at] = value

    put(0, 1, math.inf)    # slopes of 0.5: a weight of e^-350, 0 in 32 bits
    put(1, 2, math.nan)
    put(690, 3, -math.inf)
    put(691, 4, math.inf)
    put(692, 4, -math.inf)
    cache = PagedCache(*(t.to(device) for t in (keys, values, table)),
                       torch.tensor([n], dtype=torch.int32, device=device))
    query = torch.randn(1, 6, dim, generator=gen).bfloat16().to(device)
    slopes = torch.full((6,), 0.5, device=device)
    nan, inf = {1, 2, 4}, {3}
    for options, nans in ((dict(slopes=slopes), nan), (dict(slopes=slopes, softcap=20.0), nan),
                          (dict(softcap=20.0), {2, 4}), (dict(window=100), {4}),
                          (dict(window=100, slopes=slopes), {4}), ({}, {2, 4})):
        got = paged_decode(query, cache, backend=backend, **options).cpu()[0]
        # (without slopes the first token weighs something: its infinity is one)
        infs = inf | ({1} if "slopes" not in options and "window" not in options else set())
        for d in range(dim):
            want = "nan" if d in nans else "inf" if d in infs else "finite"
            kind = [("nan" if v != v else "inf" if math.isinf(v) else "finite")
                    for v in got[:, d].float().tolist()]
            assert kind == [want] * 6, (d, options)
        assert bool((got[:, 3] == -math.inf).all())


def test_torch():
    check("cpu", "auto")


@pytest.mark.gpu
def test_hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    check("cuda", "hip")
