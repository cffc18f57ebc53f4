"""tests/cpp/test_int8: the C++ host API's operators in 8-bit integers."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(suite: str) -> str:
    path = os.path.join(ROOT, "tests", "cpp", "_build", "test_int8")
    if not os.path.exists(path):
        pytest.fail(f"{path} is missing: build it with __graft_entry__.build()")
    result = subprocess.run([path, suite], capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, result.stdout + result.stderr
    return result.stdout


def test_cpp_int8_sizes():
    assert "i8_rows_lie_at_multiples_of_16 ... ok" in _run("cpu")


@pytest.mark.gpu
def test_cpp_int8_products_and_refusals():
    out = _run("gpu")
    for name in ("i8_calls_refuse_by_fault", "i8_products_in_a_graph"):
        assert name + " ... ok" in out
