"""Bounded waits of the kernels, read from their sources (a wait that runs out is not staged on a GPU): a warp that goes on to warp-wide
instructions asks as a whole whether its wait succeeded.  Lanes that answered for themselves could part ways when a limit passes, some
leaving and some waiting for them without a limit."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "sm120-nvfp4-training_b200" / "csrc"


def calls(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    return [text[max(0, m.start() - 60):text.index(";", m.end()) + 80] for m in re.finditer(r"\bmbar_wait\(", text)]


@pytest.mark.parametrize("name", ["gemm.cu", "fp8_gemm.cu"])
def test_tensor_core_kernels_wait_by_the_warp(name):
    assert calls(name) == []
    assert (CSRC / name).read_text().count("mbar_wait_warp(") >= 4


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cu")))
def test_waits_that_decide_the_way_are_asked_by_the_warp(name):
    for call in calls(name):
        decides = re.search(r"\b(if|while|return)\b[^;{]*mbar_wait\(|=\s*(__all_sync\([^;]*)?mbar_wait\(", call)
        assert not decides or "__all_sync" in call, call
