"""Resources of the built paged-cache and rotary kernels (nothing is launched;
the code objects are this repository's own)."""

import re

from test_kernel_resources_cpu import kernels, needs_tools  # noqa: F401


def _family(kernels, name):  # noqa: F811
    found = {k: v for k, v in kernels.items() if re.search(r"\d" + name, k)}
    assert found, name
    return found


@needs_tools
def test_every_dim_and_type_is_built_without_scratch(kernels):  # noqa: F811
    for family in ("paged_kernel", "paged_join_kernel"):
        found = _family(kernels, family)
        args = {re.search(family + r"ILi(\d+)ELb([01])E", k).groups() for k in found}
        assert args == {(str(d), h) for d in range(32, 257, 32) for h in "01"}
        for name, res in found.items():
            assert res["spill"] == 0 and res["scratch"] == 0, (name, res)
    for name, res in _family(kernels, "rotary_kernel").items():
        assert res["spill"] == 0 and res["scratch"] == 0, (name, res)
