"""Resources of the built kernels of the 4-bit cache and of prompts (nothing is
launched; the code objects are this repository's own)."""

import re

from test_kernel_resources_cpu import kernels, needs_tools  # noqa: F401
from test_paged_resources_cpu import _family

DIMS = {str(d) for d in range(32, 257, 32)}


@needs_tools
def test_every_dim_type_and_form_is_built(kernels):  # noqa: F811
    for family in ("quantized_kernel", "prompt_kernel", "paged_kernel"):
        found = _family(kernels, family)
        args = {re.search(family + r"ILi(\d+)ELb([01])ELb([01])E", k).groups() for k in found}
        assert args == {(d, half, scores) for d in DIMS for half in "01" for scores in "01"}
    for family in ("prompt_join_kernel", "paged_join_kernel"):
        args = {re.search(family + r"ILi(\d+)ELb([01])E", k).groups()
                for k in _family(kernels, family)}
        assert args == {(d, half) for d in DIMS for half in "01"}
    # (the prompt kernel's registers are full from head_dim 96 on: what it spills are
    # addresses and bounds outside its products)
    for family in ("quantized_kernel", "quantize_rows_kernel", "quantized_read_kernel",
                   "paged_read_kernel", "prompt_join_kernel"):
        for name, res in _family(kernels, family).items():
            assert res["spill"] == 0 and res["scratch"] == 0, (name, res)
    for name, res in _family(kernels, "prompt_kernel").items():
        assert res["lds"] <= 80 * 1024, (name, res)  # two workgroups on a CU
