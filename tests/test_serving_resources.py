"""No kernel of the serving operators uses scratch or spills vector registers (read from the built code objects)."""

import pytest

from tests.test_kernel_resources import BUILD, _kernels


@pytest.mark.parametrize("src", ["tsfa_append", "tsfa_beam", "tsfa_varlen"])
def test_no_scratch(src):
    kernels = _kernels(BUILD / f"{src}.o")
    assert kernels, f"no kernels found in {src}.o"
    for name, k in kernels.items():
        assert k.get("private_segment_fixed_size", 0) == 0, f"{name} uses scratch"
        assert k.get("vgpr_spill_count", 0) == 0, f"{name} spills VGPRs"
