"""Rules that the kernels' sources keep, checked on the text: no GPU needed."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "spmd-dialect_b200" / "csrc"
OVERLAPPING = ["layer_norm.cu", "layer_norm_backward.cu", "grad_norm.cu", "reduce.cu", "reduce_kinds.cu"]


def kernels_of(text: str):
    """(signature, body) of every __global__ function."""
    for m in re.finditer(r"^__global__[^{;]*\{", text, re.M):
        end = text.index("\n}\n", m.end())
        yield m.group(0), text[m.end():end]


@pytest.mark.parametrize("name", OVERLAPPING)
def test_kernels_that_overlap_promise_nothing_about_memory(name):
    """A kernel that may start before the one that writes its input has ended must not declare the input as read-only
    for its own lifetime (const ... __restrict__): its loads could leave their place behind the wait."""
    waiting = [(sig, body) for sig, body in kernels_of((CSRC / name).read_text()) if "pdl_wait()" in body]
    assert waiting
    for sig, body in waiting:
        assert "__restrict__" not in sig and "__ldg" not in body, sig.split("(")[0]
