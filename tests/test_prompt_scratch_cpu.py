"""Registers of the built prompt kernels that live in scratch (nothing is launched;
the code objects are this repository's own)."""

import re

from test_kernel_resources_cpu import kernels, needs_tools  # noqa: F401
from test_paged_resources_cpu import _family

# bytes a lane, at most: up to head_dim 128 two waves a SIMD have 256 registers each (at
# 128 nothing of it is in the loop over tiles), behind it one has 512, and at 256 the
# query's 64, the accumulators' 128 and a tile's leave no room for all (28 of the
# query's are read again beside each tile's products)
SCRATCH = {128: 68, 224: 96, 256: 272}


@needs_tools
def test_scratch_of_the_prompt_kernels(kernels):  # noqa: F811
    for name, res in _family(kernels, "prompt_kernel").items():
        most = SCRATCH.get(int(re.search(r"prompt_kernelILi(\d+)E", name)[1]), 0)
        assert res["scratch"] <= most, (name, res)
