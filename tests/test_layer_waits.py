"""Waits of whole warps: what follows them in a kernel is the warp's (products, shuffles, copies of one elected lane), so its lanes have to leave a wait together and with one answer."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy3_b200", "csrc")


@pytest.mark.parametrize("file", ["linear4.cu", "linear4_umma.cu", "experts_umma.cu"])
def test_no_lane_waits_by_itself(file):
    with open(os.path.join(CSRC, file)) as f:
        text = f.read()
    assert len(re.findall(r"\bwarp_wait\(", text)) >= 3
    assert not re.findall(r"\bmbar_(?:wait|try)\(", text.replace("__all_sync(0xffffffffu, mbar_wait(", ""))
    # nor does a warp's loop end by what its lanes read of the abort flag one by one
    assert not re.findall(r"for \([^;]*;[^;]*\*s_abort", text)


def test_adapters():
    """Its copies and products are one lane's, which waits alone; the warps that store results wait as warps."""
    with open(os.path.join(CSRC, "adapters.cu")) as f:
        text = f.read()
    assert re.findall(r"\b(mbar|warp)_wait\([^;]*A_(\w+) \+", text) == [("mbar", "EMPTY"), ("mbar", "EMPTY"), ("mbar", "TEMPTY"), ("mbar", "FULL"), ("warp", "TFULL")]


@pytest.mark.gpu
@pytest.mark.parametrize("which,where", [(0, 29), (1, 39), (4, 49)])
def test_a_warp_whose_lanes_saw_different_phases_gives_up_as_one(cuda, which, where):
    """Lane 0 asks for a phase that is over, the others for one that nothing ends: if lane 0 went on, another place would be reported."""
    import torch
    import hy3_b200
    hy3_b200.layer_sync()
    assert hy3_b200.load_library().hy3a_layer_wait_out(torch.cuda.current_stream().cuda_stream, which) == 0
    with pytest.raises(hy3_b200.Hy3AttnError, match=r"where %d\)" % where):
        hy3_b200.layer_sync()
    hy3_b200.layer_sync()
