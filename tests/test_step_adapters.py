"""include/fqa_step.hpp's adapter calls on the host, the device stubbed out, under AddressSanitizer +
UndefinedBehaviorSanitizer (tests/cpp/step_adapters_host.cpp): whatever batch is uploaded, the bounds that
fqa_lora_plan is given are within the context's buffers."""
from __future__ import annotations

import pytest

from tests.test_sanitize import CLANG, _build, _run

pytestmark = pytest.mark.skipif(not CLANG.exists(), reason="ROCm clang not present")


def test_plans_stay_within_the_contexts_buffers():
    exe = _build("step_adapters_host", ["tests/cpp/step_adapters_host.cpp", "oracle/fqa_oracle.c"], cxx=True)
    assert _run(exe).strip() == "ok"
