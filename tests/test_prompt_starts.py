"""Starts of prompts' rows that decrease: no row is any sequence's."""

import pytest
import torch

from refinekv import PagedCache, paged_prompt, prompt_attention

BF16 = torch.bfloat16
# 8 rows, of which the last comes again and again
AGAIN = [0, 8] + [7, 8] * 20


def check(device, backend):
    gen = torch.Generator().manual_seed(1)
    query = torch.randn(8, 256, 64, generator=gen).to(BF16).to(device)
    keys = [torch.randn(3000, 1, 64, generator=gen).to(BF16).to(device) for _ in range(2)]
    pages = [t.view(-1, 1, 50, 64)[:8, :, :16].contiguous() for t in keys]
    for starts in (AGAIN, [0, 8, 3, 8], [8, 0], [0, 3] * 200, [5, 2, 2 ** 31 - 1],
                   [0, 8] + [8] * 300 + [7]):
        count = len(starts) - 1
        at = torch.tensor(starts, dtype=torch.int32, device=device)
        ends = torch.full((count + 1,), 3000, dtype=torch.int32, device=device)
        ends[::2] = 0
        cache = PagedCache(*pages, torch.zeros(count, 5, dtype=torch.int32, device=device),
                           torch.full((count,), 70, dtype=torch.int32, device=device))
        calls = (lambda **k: prompt_attention(query, *(t[:8] for t in keys), token_starts=at,
                                              backend=backend, **k),
                 lambda **k: prompt_attention(query, *keys, token_starts=at, key_starts=ends,
                                              backend=backend, **k),
                 lambda **k: paged_prompt(query, cache, token_starts=at, backend=backend, **k))
        for call in calls:
            poison = torch.full_like(query, 7.0)  # (memory that the new tensor may take)
            del poison
            assert not bool(call().any()), starts[:4]
            kept = torch.full_like(query, 7.0)
            call(output=kept)
            assert bool((kept == 7.0).all()), starts[:4]
    # equal ones are empty sequences
    at = torch.tensor([0, 0, 5, 5, 8, 8], dtype=torch.int32, device=device)
    few = [t[:8] for t in keys]
    got = prompt_attention(query, *few, token_starts=at, backend=backend)
    for part in (slice(0, 5), slice(5, 8)):
        alone = prompt_attention(query[part], *(t[part] for t in few), backend=backend)
        assert torch.equal(got[part], alone)


def test_torch():
    check("cpu", "auto")


@pytest.mark.gpu
def test_hip():
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    check("cuda", "hip")
