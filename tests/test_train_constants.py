"""Constants that the Python side repeats agree with the library's.  No GPU needed."""
from __future__ import annotations

import re

from conftest import ROOT, spmd_mod


def test_held_columns():
    held, size = spmd_mod("kernels").HELD_COLUMNS, spmd_mod("_lib").lib().spmdb200_layer_norm_forward_workspace_bytes
    assert size(1000, held) == 0 and size(1000, held + 1) > 0
    text = (ROOT / "include" / "spmd_b200.h").read_text()
    assert re.search(rf"0 bytes \(NULL\) for rows of up to {held} elements", text)


def test_state_block_and_types():
    k, text = spmd_mod("kernels"), (ROOT / "include" / "spmd_b200.h").read_text()
    macros = dict(re.findall(r"^#define SPMDB200_(\w+) (\d+)$", text, re.M))
    assert int(macros["STATE_BLOCK"]) == k.STATE_BLOCK
    assert {str(t).split(".")[1]: c for t, c in k._TYPES.items()} == {
        "float32": int(macros["F32"]), "float16": int(macros["F16"]), "bfloat16": int(macros["BF16"])}
