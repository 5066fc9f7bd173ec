"""CPU: what the 8-bit rows' kernels keep to, read from their sources."""
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "vila_b200" / "csrc"


@pytest.mark.parametrize("name", ["fp8.cuh", "fp8.cu", "fp8_linear.cu", "fp8_tc.cu", "fp8_pair.cu"])
def test_nothing_is_read_by_the_read_only_path(name):
    """These kernels begin while the launch before may still write their inputs: loads that take them for constant during the whole launch are
    neither ordered behind the wait for that launch nor bound to the condition around them."""
    text = (CSRC / name).read_text()
    assert "__ldg" not in text and "ld.global.nc" not in text and "ldg_stream" not in text
