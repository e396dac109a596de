"""tests/cpp/adapters_graph_cpp.cpp: a step with adapters captured by the C++ step context's bounds and
replayed for other batches, bf16 and fp32, checked in the program itself in whole numbers."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.gpu
def test_adapters_in_a_captured_step(gpu):
    exe = ROOT / "tests" / "cpp" / "adapters_graph_cpp"
    if not exe.exists():
        from flashqwen_amd import build

        build.build_adapters_driver()
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    print(r.stdout, flush=True)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr
