"""What `make` builds, read from its plan (nothing is compiled)."""
import os
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yolo_from_scratch_amd", "csrc")


def _plan(python):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, f"PYTHON={python}"], check=True, capture_output=True, text=True).stdout


def test_library_needs_no_torch():
    """The C library is built by a plain `make` where no torch is installed; the extension module, which needs torch's headers, is
    left out with a word.  With torch both are built."""
    without = _plan("true")                       # an interpreter that finds nothing
    assert "../libyfs.so" in without and "torch_binding.cpp" not in without and "_binding.so" in without
    both = _plan(sys.executable)
    assert "../libyfs.so" in both and "torch_binding.cpp -o ../_binding.so" in both


def test_extension_module_refuses_an_older_library(monkeypatch):
    from types import SimpleNamespace
    from yolo_from_scratch_amd import _lib as L
    monkeypatch.setattr(L, "_binding", None)
    monkeypatch.setattr(L, "_lib", SimpleNamespace(yfs_version=lambda: 300))
    with pytest.raises(L.YfsError, match="version 300"):
        L.binding()
