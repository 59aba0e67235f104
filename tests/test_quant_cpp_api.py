"""Runs the C++ test of the quantised serving operators (tests/cpp/test_quant_api.cpp, built by build())."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

BIN = Path(__file__).resolve().parent / "cpp" / "_build" / "test_quant_api"


def _run(*args):
    assert BIN.exists(), f"{BIN} is missing: run __graft_entry__.build() first"
    res = subprocess.run([str(BIN), *args], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    print(res.stdout)
    assert res.returncode == 0 and " 0 failed" in res.stdout, res.stdout


def test_cpp_quant_api_cpu():
    _run("--cpu")


@pytest.mark.gpu
def test_cpp_quant_api_gpu():
    _run()
