"""tests/cpp/test_tree: the C++ host API's operators on trees of drafted tokens."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(suite: str) -> str:
    path = os.path.join(ROOT, "tests", "cpp", "_build", "test_tree")
    if not os.path.exists(path):
        pytest.fail(f"{path} is missing: build it with __graft_entry__.build()")
    result = subprocess.run([path, suite], capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stdout + result.stderr
    return result.stdout


def test_cpp_tree_masks():
    assert "tree_masks_hold_ancestors ... ok" in _run("cpu")


@pytest.mark.gpu
def test_cpp_tree_step_and_refusals():
    out = _run("gpu")
    for name in ("tree_calls_refuse_by_fault", "tree_step_in_a_graph"):
        assert name + " ... ok" in out
