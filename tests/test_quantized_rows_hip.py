"""Rows of the append to a 4-bit cache that are views of its tensors (GPU)."""

import pytest
import torch

from refinekv import QuantizedCache, Rotary, RotaryConfig, paged_append

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


@pytest.mark.parametrize("part", ["key_codes", "value_codes", "key_scales", "value_scales"])
def test_views_that_a_call_would_copy_are_refused(part):
    """At odd addresses, and with dims apart: the kernel does not take them, and a
    copy would hide what they are."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    cache = QuantizedCache.empty(64, 2, 16, 64, 3, 2, device=DEV)
    pool = getattr(cache, part).view(-1).view(BF16)
    rows = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    rotary = Rotary(RotaryConfig(head_dim=64), DEV)
    for inside in (pool[:384].view(3, 2, 64), pool[1:385].view(3, 2, 64),
                   pool[:768].view(3, 2, 64, 2)[..., 0],
                   pool[-400:].as_strided((3, 2, 64), (130, 65, 1))):
        for name in ("key", "value", "query"):
            args = dict(key=rows, value=rows, query=rows, rotary=rotary)
            with pytest.raises(ValueError, match="overlap the cache"):
                paged_append(**{**args, name: inside}, cache=cache, backend="hip")
    # rows elsewhere at such places are copied, as before
    store = torch.zeros(800, dtype=BF16, device=DEV)
    for apart in (store[1:385].view(3, 2, 64), store[:768].view(3, 2, 64, 2)[..., 0]):
        paged_append(apart, apart, cache, query=apart, rotary=rotary, backend="hip")
