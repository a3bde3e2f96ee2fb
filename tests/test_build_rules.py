"""The Makefile's rules, without running them."""
import os
import subprocess
import sys

import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rgpt_b200", "csrc")


def plan(*args):
    r = subprocess.run(["make", "-n", "-C", CSRC, *args], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


def test_kernels_build_without_torch_or_python_headers():
    for python in ("false", f"{sys.executable} -S"):  # no interpreter; one that finds no torch
        out = plan("-B", f"PYTHON={python}")
        assert "-c gemm.cu" in out and "fastargs.cpp" not in out


def test_argument_checks_are_built_again_for_another_torch():
    python = f"PYTHON={sys.executable}"
    assert "fastargs.cpp" in plan("-B", python)
    as_they_are = ("-o", "Makefile", "-o", "fastargs.cpp", python)
    if os.path.exists(os.path.join(CSRC, "..", "_fastargs.so")):
        assert "fastargs.cpp" not in plan(*as_they_are)
    version = os.path.join(os.path.dirname(torch.__file__), "version.py")
    assert "fastargs.cpp" in plan("-W", version, *as_they_are)
