"""FP8 expert layers through the C++20 host layer: the test program tests/cpp/test_fp8.cpp (built by
__graft_entry__.build() via tests/cpp/Makefile)."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

BIN = Path(__file__).resolve().parent / "cpp" / "_bin" / "test_fp8"


def _run(mode: str) -> None:
    assert BIN.exists(), f"{BIN} is not built: run __graft_entry__.build()"
    res = subprocess.run([str(BIN), mode], capture_output=True, text=True, timeout=100)
    print(res.stdout, res.stderr)
    assert res.returncode == 0 and " 0 failures" in res.stdout, res.stdout + res.stderr


def test_cpp_fp8_cpu():
    _run("cpu")


@pytest.mark.gpu
def test_cpp_fp8_gpu():
    print("[gpu] C++ FP8 layer", flush=True)
    _run("gpu")
