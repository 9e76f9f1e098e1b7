"""What the operators around the routed experts promise, as far as it shows without a GPU."""
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crosslane_b200", "csrc")


@pytest.mark.parametrize("name", ["clb_route.cu", "clb_block_norm.cu", "clb_int8.cu", "clb_ops.cuh", "clb_tc.cuh"])
def test_kernels_set_up_early_read_coherently(name):
    """A kernel whose CTAs start under the end of the one in front must not read what that one writes through the
    read-only path, whose data has to stay constant for the kernel's life."""
    with open(os.path.join(CSRC, name)) as f:
        code = "".join(line.split("//")[0] for line in f)
    assert "__ldg" not in code and "ld.global.nc" not in code and "__restrict__" not in code
