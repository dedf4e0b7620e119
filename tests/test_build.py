"""What `make` and build() make, asked of make itself without running it."""
import os
import subprocess
import sys

import __graft_entry__ as entry

CSRC = os.path.join(entry.ROOT, "multimodal_transformer_amd", "csrc")


def _would_run(*args):
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], check=True, capture_output=True, text=True).stdout


def test_the_library_needs_no_torch():
    """Without a Python that has torch the default target is the library alone."""
    with_torch, without = _would_run(f"PYTHON={sys.executable}"), _would_run("PYTHON=/bin/false")
    assert "libmmt_amd.so" in with_torch and "_autograd.so" in with_torch
    assert "libmmt_amd.so" in without and "_autograd.so" not in without
    assert "_autograd.so" in _would_run("PYTHON=/bin/false", "autograd")


def test_build_compiles_what_is_built_already(monkeypatch):
    seen = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd: seen.append(cmd))
    entry.build()
    assert seen and "-B" in seen[0] and {"all", "autograd"} <= set(seen[0])
