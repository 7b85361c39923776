"""Batches of drafted trees through the C++ host interface (moa-workspace_amd/host/moa_ops.hpp) without max_rows: their harness,
tests/cpp/test_tree_batches, compares them with calls that say it."""
import subprocess
from pathlib import Path

import pytest

HARNESS = Path(__file__).resolve().parent / "cpp" / "test_tree_batches"


def run():
    if not HARNESS.exists():
        pytest.fail(f"{HARNESS} is not built (run __graft_entry__.build())")
    return subprocess.run([str(HARNESS)], capture_output=True, text=True, timeout=100)


@pytest.mark.gpu
def test_the_harness_passes():
    from gpu_util import need_gpu, say
    need_gpu()
    say("C++ batches of trees")
    res = run()
    print(res.stdout, flush=True)
    assert res.returncode == 0, res.stdout + res.stderr
    lines = [line.rstrip() for line in res.stdout.splitlines()]
    assert sum(line.endswith("-> PASS") for line in lines) == 5
    assert lines[-1] == "PASS: 0 checks failed"


def test_without_a_device_it_fails_with_the_librarys_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is visible")
    res = run()
    assert res.returncode == 1, res.stdout + res.stderr
    assert "FAIL:" in res.stdout and "code" in res.stdout, res.stdout
