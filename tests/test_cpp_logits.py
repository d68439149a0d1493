"""Runs the C++ programs for rows of logits (tests/cpp/test_raft_logits*.cpp): refusals without a
GPU; top_k, distillation and sampling through a handle on the GPU."""
import subprocess
from pathlib import Path

import pytest

BIN = Path(__file__).resolve().parent / "cpp" / "bin"


def _run(name, timeout):
    exe = BIN / name
    if not exe.exists():
        from raft_amd import build
        build.build_cpp_tests()
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=timeout)
    tail = "\n".join(proc.stdout.splitlines()[-40:])
    assert proc.returncode == 0, f"{name} failed (rc={proc.returncode}):\n{tail}\n{proc.stderr[-2000:]}"
    assert "0 failed" in proc.stdout


def test_cpp_logits_refusals():
    _run("test_raft_logits_host", 60)


@pytest.mark.gpu
def test_cpp_logits_on_gpu(gpu):
    _run("test_raft_logits", 100)
