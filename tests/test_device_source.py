"""What the device sources must keep to and no run can show: a fault there
would need a lane-by-lane race with the clock."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "python-gen-worker_b200" / "csrc"


@pytest.mark.parametrize("name", ["gated.cu", "gemm.cu"])
def test_epilogue_waits_take_the_whole_warp(name):
    """Accumulator loads need every lane of the warp. A bounded wait may run out
    in some lanes and not in others, so a role that reads accumulators must
    leave its loop as a warp: it waits by the form that votes."""
    waits = re.findall(r"(mbar_wait\w*)\([^;]*?GWB_ERR_TIMEOUT_EPILOGUE\)",
                       (CSRC / name).read_text())
    assert waits and set(waits) == {"mbar_wait_warp"}
