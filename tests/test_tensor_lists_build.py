"""The native reader of tensor lists: loaded by the functions that need it, and
rebuilt when torch or Python changes.  No GPU needed."""
from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import ROOT, spmd_mod

PROGRAM = """
import importlib, sys
name = "spmd-dialect_b200._tensor_lists"
{before}
kernels = importlib.import_module("spmd-dialect_b200.kernels")
importlib.import_module("spmd-dialect_b200.shard")
{after}
"""


def run(before: str, after: str) -> str:
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(before=before, after=after)], cwd=ROOT, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_the_other_kernels_do_not_load_the_reader():
    run("", "assert name not in sys.modules")


def test_without_the_reader_only_lists_fail():
    """A module built against another torch, or not built: the list functions say so, nothing else is affected."""
    out = run("sys.modules[name] = None", """
import torch
for call in (lambda: kernels._read_list("grad_norm", [], 0, 1, None), ):
    try:
        call()
    except ImportError as e:
        print(e)
try:
    kernels.layer_norm(torch.ones(2, 8))
except ValueError:
    print("refused as before")
""")
    assert "build.py" in out and "refused as before" in out


def test_reader_is_found_at_its_first_use():
    run("", """
p, s, t = kernels._read_list("list", [], 0, 1, None)
assert (p, s, t) == (b"", b"", b"") and name in sys.modules
assert kernels._read_list("list", [], 0, 1, None) == (b"", b"", b"")
""")


@pytest.fixture
def build(tmp_path, monkeypatch):
    b = spmd_mod("build")
    monkeypatch.setattr(b, "LISTS", tmp_path / "_tensor_lists.so")
    monkeypatch.setattr(b, "LISTS_FOR", tmp_path / "tensor_lists.for")
    commands = []

    def fake(cmd):
        commands.append(cmd)
        b.LISTS.write_bytes(b"")
        return ""

    monkeypatch.setattr(b, "_run", fake)
    b.commands = commands
    return b


def test_reader_is_rebuilt_for_another_torch(build, monkeypatch):
    import torch
    assert build.lists_stale()
    build.build_lists()
    assert len(build.commands) == 1 and not build.lists_stale()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.lists_stale()
    build.build_lists()
    assert not build.lists_stale()
    build.LISTS_FOR.unlink()
    assert build.lists_stale()


def test_no_torch_no_reader(build, monkeypatch):
    """The library itself needs no torch: without one there is nothing to read lists of."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert not build.lists_stale()


def test_written_raises_versions():
    run("", """
import torch
kernels._read_list("list", [], 0, 1, None)
a, b = torch.ones(3), torch.ones(5)
with torch.inference_mode():
    c = torch.ones(2)
kernels._written([a, None, b, c], None, [a])
assert a._version == 2 and b._version == 1
try:
    kernels._written((a,))
except TypeError:
    assert a._version == 2
""")
