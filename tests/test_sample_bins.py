"""What fqa_sample_filtered's scan computes of its bins (flashqwen_amd/csrc/fqa_sample_bins.h), run on
the host by tests/cpp/sample_bins.cpp, built with UndefinedBehaviorSanitizer."""
from __future__ import annotations

import math
import re
import subprocess

import pytest

from tests.test_sanitize import CLANG, ENV, ROOT

pytestmark = pytest.mark.skipif(not CLANG.exists(), reason="ROCm clang not present")


@pytest.fixture(scope="module")
def bins(tmp_path_factory):
    exe = tmp_path_factory.mktemp("bins") / "sample_bins"
    subprocess.run([str(CLANG) + "++", "-O1", "-g", "-std=c++17", "-Wall", "-ffp-contract=off",
                    "-fsanitize=undefined", "-fno-sanitize-recover=all", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", str(ROOT / "tests" / "cpp" / "sample_bins.cpp"), "-o",
                    str(exe)], check=True, capture_output=True, text=True)

    def run(*args):
        r = subprocess.run([str(exe), *args], capture_output=True, text=True, env=ENV, timeout=120)
        assert r.returncode == 0, (r.returncode, r.stdout[-500:], r.stderr[-2000:])
        return r.stdout

    return run


def test_slots_of_far_places(bins):
    """Places up to 2^30: no term of a histogram index leaves its type."""
    n = int(bins("slots").split()[0])
    assert n > 100 * 384 * 4, n


def test_weights_are_as_close_as_the_header_says(bins):
    """The scan's weights against exp2 in 64 bits of significand: within what fqa.h states of them, and
    not closer than a quarter of that (a stated bound is one that the code has)."""
    text = (ROOT / "include" / "fqa.h").read_text()
    stated = 2.0 ** -int(re.search(r"Weights are held to[\s*]+2\^-(\d+) of their value", text).group(1))
    worst = float(bins("weights"))
    print(f"worst relative error {worst:.3g} = 2^{math.log2(worst):.2f}, stated {stated:.3g}")
    assert stated / 4 < worst <= stated
