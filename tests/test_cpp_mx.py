"""Layer norm and MXFP4 through the C++ host layer: tests/cpp/mx_layer_norm_test checks its results itself."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "mx_layer_norm_test")


def run(what):
    out = subprocess.run([BIN, what], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr + out.stdout
    assert f"{what} ok" in out.stdout


def test_cpp_sizes_and_refusals():
    if not os.path.exists(BIN):
        subprocess.check_call(["make", "-s", "-C", os.path.dirname(BIN)])
    run("cpu")


@pytest.mark.gpu
def test_cpp_layer_norm_and_mxfp4_on_gpu():
    assert os.path.exists(BIN), "tests/cpp/mx_layer_norm_test has not been built (run __graft_entry__.build())"
    run("gpu")
