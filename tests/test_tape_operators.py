"""The long-history operators on the C++ device tape: tests/cpp/test_tape_operators (built by __graft_entry__.build())."""
import os
import subprocess

import pytest

import talos_hip as th

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_tape_operators")


def _run():
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} is missing: run __graft_entry__.build()")
    return subprocess.run([BIN], capture_output=True, text=True, timeout=110)


@pytest.mark.gpu
def test_operators_on_the_tape():
    r = _run()
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
    assert " 0 failed" in r.stdout


def test_operators_on_the_tape_without_gpu_fail_cleanly():
    if th.device_count() > 0:
        pytest.skip("a GPU is present")
    r = _run()
    assert r.returncode == 1
    assert "no usable GPU" in r.stdout
