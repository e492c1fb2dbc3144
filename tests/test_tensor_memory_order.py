"""Tensor memory is taken before the next kernel is let in.  A kernel that is let in holds its columns while it waits for the one in front, whose
allocation has no bound: where both do not fit, each would wait for the other."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "gguf2bin_b200" / "csrc"


def calls(text):
    """The order of the calls of a source: 'take' (tmem_alloc, tmem_alloc_pair) and 'let in' (pdl_launch); comments are none."""
    text = re.sub(r"//[^\n]*", "", text)
    return [("take" if m.group(1).startswith("tmem") else "let in") for m in re.finditer(r"\b(tmem_alloc(?:_pair)?|pdl_launch)\(", text)]


@pytest.mark.parametrize("unit", ["gemm_fp8_few.cuh", "gemm_fp8_tc.cuh", "attn_prefill_tc_split.cu"])
def test_who_takes_before_it_lets_in(unit):
    order = calls((CSRC / unit).read_text())
    assert order == ["take", "let in"]

