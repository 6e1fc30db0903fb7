"""The paged decode's softmax weights enter the second product whole (GPU).

An output that rounds to its type hides an error of its weights, unless large
terms cancel: two visible values of +1 and -1 with nearly the same weight leave
an output a thousand times smaller than either term.
"""

import pytest
import torch

from paged_math import half_step, tiny
from refinekv import PagedCache, paged_decode

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [32, 128])
def test_cancelling_values_show_whole_weights(dtype, dim):
    """400 sequences of three tokens: one with the largest score and value 0,
    two whose scores differ by 2^-14 and whose values are +1 and -1.  A score
    is the sum of a key's first two dims, exact in fp32.

    Room.  In units of 2^-24, a weight e^-|x| (|x| <= 1) is off by: the folded
    scale 1 |x|, the product with it 1 |x|, the difference to the maximum 1 |x|
    (ln 2 of it once in base 2, below 1), the hardware's 2^x 2, its parts' sum 2
    (fp16: two parts reach 2^-23; bf16: three are exact), so at most 7 of each
    of the two weights; the products' sums and the division add 4 of their
    size, which is below one weight.  Divided by a sum of at least 1 + 2 w, the
    two weights give less than 7 + 4 in all.  Then the result, of about 2^-16,
    is rounded to the type."""
    gen = torch.Generator().manual_seed(dim)
    count, page = 400, 16
    low = -torch.rand(count, generator=gen).clamp_min(0.1).to(dtype).double()
    keys = torch.zeros(count, 1, page, dim, dtype=torch.float64)
    values = torch.zeros_like(keys)
    keys[:, 0, 1:3, 0] = low[:, None]
    keys[:, 0, 2, 1] = 2.0 ** -14
    values[:, 0, 1], values[:, 0, 2] = 1.0, -1.0
    scores = keys[:, 0, :3].sum(-1)
    want = torch.softmax(scores, -1) @ torch.tensor([0.0, 1.0, -1.0], dtype=torch.float64)
    assert torch.equal(keys.to(dtype).double(), keys)
    query = torch.zeros(count, 1, dim, dtype=dtype)
    query[..., :2] = 1.0
    cache = PagedCache(keys.to(dtype).to(DEV), values.to(dtype).to(DEV),
                       torch.arange(count, dtype=torch.int32, device=DEV)[:, None].contiguous(),
                       torch.full((count,), 3, dtype=torch.int32, device=DEV))
    got = paged_decode(query.to(DEV), cache, scaling=1.0, backend="hip").cpu().double()
    error = (got - want[:, None, None]).abs()
    room = 11 * 2.0 ** -24
    room += half_step(dtype) * (want.abs() + room) + tiny(dtype)
    worst = float((error - room[:, None, None]).max())
    assert worst <= 0, f"{float(error.max()):.2e} off, {worst:.2e} more than rounding explains"
    assert bool(got.isfinite().all())
