"""lora_add at the edges of what it takes: plans over adapters that the weights lack."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_lora import _case, _check, _meta, _run, _t, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f32", [False, True])
def test_new_tensor_holds_y_in_every_row(gpu, f32):
    """Without `out`, rows of adapters that the weights lack and rows that the plan does not hold are
    y's: a plan serves projections whose weights hold different adapters."""
    import torch

    from flashqwen_amd.lora import lora_plan

    rng = np.random.default_rng(21)
    c = _case(rng, [3, 1, 140, 1, 2], 2, 16, 128, (64, 64), f32, none=0.0)
    ids = np.array([0, 5, 1, 7, -1], np.int32)
    T, held = c["T"], c["T"] - 2  # the plan leaves the last request out
    plan = lora_plan(_t(ids), _t(c["cu"]), _meta(4, held), 9, held)
    c["ids"] = np.where(ids < 2, ids, -1).astype(np.int32)
    want, err = _want(c)
    y = c["y"].cuda()
    keep = y.clone()
    junk = torch.full_like(y, 7.0)  # what the allocator hands out next
    del junk
    got = _run(c, plan, y=y)
    _check(got, want, err, f32, "new tensor")
    theirs = torch.from_numpy(np.repeat(c["ids"], np.diff(c["cu"])) < 0).to(gpu)
    assert torch.equal(got[theirs], y[theirs]) and torch.equal(y, keep)
    # y with a row stride, and a single row
    wide = torch.full((T, 128 + 8), 3.0, dtype=y.dtype, device=gpu)
    wide[:, :128] = y
    assert torch.equal(_run(c, plan, y=wide[:, :128]), got)
    one = lora_plan(_t(ids[1:2]), _t(np.array([0, 1], np.int32)), _meta(1, 1), 9, 1)
    assert torch.equal(_run(c, one, y=y[:1], x=c["x"][:1].cuda()), y[:1])
