"""What QuantizedCache.packed and empty take: codes of 4 bits, scales as the
kernels' products hold them exactly, whole groups."""

import math

import pytest
import torch

from refinekv import QuantizedCache, quantized

F16 = torch.float16


def parts(device, dim=64):
    gen = torch.Generator().manual_seed(dim)
    found = [quantized.quantize(torch.randn(2, 3, 16, dim, generator=gen)) for _ in range(2)]
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    return [t.to(device) for t in (found[0][0], found[1][0], found[0][1], found[1][1], table,
                                   lengths)]


def packed_with(device, which, place, value):
    args = parts(device)
    args[which][place] = value
    return QuantizedCache.packed(*args, dtype=F16)


@pytest.mark.parametrize("which", [0, 1])
def test_codes_are_of_4_bits(which):
    packed_with("cpu", which, (1, 2, 7, 40), 15)
    for code in (16, 200):
        with pytest.raises(ValueError, match="codes"):
            packed_with("cpu", which, (1, 2, 7, 40), code)


def test_head_dims_between_groups():
    for dim in (33, 48, 65, 100, 127, 257):
        with pytest.raises(ValueError, match="head_dim"):
            QuantizedCache.empty(2, 1, 16, dim, 1, 1)
    assert QuantizedCache.empty(2, 1, 16, 96, 1, 1).head_dim == 96


@pytest.mark.gpu
@pytest.mark.parametrize("which", [2, 3])
def test_scales_that_the_kernels_do_not_hold(which):
    if not torch.cuda.is_available():
        pytest.skip("no GPU in this environment")
    place = (1, 2, 7, 1, 0)  # a scale; its last index 1: a zero
    for value in (0.0, 1.0, 127.0 / 128, 544.0, 552.0, 2.0 ** -20, math.nan):
        packed_with("cuda", which, place, value)
    for value in (1.0 + 2.0 ** -7, 1.0 + 2.0 ** -10, 2.0 ** -24, -1.0, 546.0, 560.0, math.inf,
                  -math.inf):
        with pytest.raises(ValueError, match="scales"):
            packed_with("cuda", which, place, value)
    for value in (-4096.0, 1.0 / 3, math.nan):
        packed_with("cuda", which, (1, 2, 7, 1, 1), value)
    for value in (math.inf, -math.inf):
        with pytest.raises(ValueError, match="zeros"):
            packed_with("cuda", which, (1, 2, 7, 1, 1), value)
    for args in (parts("cpu"), parts("cuda")):  # as quantize gives them, rows of NaN as well
        args[2][0], args[3][1] = math.nan, math.nan
        QuantizedCache.packed(*args, dtype=F16)
