"""Runs the C++ operator layer's test programs for the 4-bit cache, the key weights and the eviction (nano-vllm-cpp_b200/host/tests/test_int4_*.cpp):
refusals without a GPU, known answers through ``Attention`` and the operators on one."""
import os
import subprocess

import pytest

from util import ROOT, entry


def _run(name):
    entry.build()
    exe = os.path.join(ROOT, "nano-vllm-cpp_b200", "build", name)
    assert os.path.exists(exe), f"{exe} was not built"
    return subprocess.run([exe], capture_output=True, text=True, timeout=300)


def test_refusals_without_a_gpu():
    res = _run("test_int4_cpu")
    assert res.returncode == 0, res.stdout + res.stderr
    assert "0 failed" in res.stdout


@pytest.mark.gpu
def test_known_answers_on_gpu():
    res = _run("test_int4_gpu")
    assert res.returncode == 0, res.stdout + res.stderr
    assert "0 failed" in res.stdout
