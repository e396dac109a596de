"""lora_add at the edges of what it takes: plans over adapters that the weights lack, infinities in the
weights, no rows at all."""
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


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T_of,R,slices", [([1, 1, 1], 16, (64,)), ([1] * 30, 32, (12224, 12352)),
                                           ([40, 300, 1], 64, (64, 256)), ([150, 9], 128, (128,))])
def test_infinities_in_the_weights(gpu, T_of, R, slices, f32):
    """An infinity of B times any h but zero is that infinity, whether h's lower parts are zero (h of
    few bits: scale 1) or not (scale 0.37); opposite ones, or one times zero, are NaN; an infinite h
    likewise."""
    import torch

    print(f"[test_infinities_in_the_weights] {T_of} R={R} {slices} f32={f32}", flush=True)
    rng = np.random.default_rng(R)
    K, n = 128, 3
    c = _case(rng, T_of, n, R, K, slices, f32, none=0.0, ranks=np.array([R, R, R - 5], np.int32))
    c["ids"] = (np.arange(len(T_of)) % n).astype(np.int32)
    c["scale"] = torch.tensor([1.0, 0.37, -1.0])
    T, N, S = c["T"], sum(slices), len(slices)
    ints = lambda m, *s: torch.from_numpy(rng.integers(-m, m + 1, s).astype(np.float32)).bfloat16()  # noqa: E731
    c["x"], c["a"], c["b"] = ints(3, T, K), ints(2, n, S * R, K), ints(5, n, N, R)
    c["a"][2, 3, 7] = float("inf")  # h[3] of the third adapter is infinite, or NaN where x[7] is 0
    for i in range(n):
        for col in range(0, N, 3):  # the columns between stay finite
            c["b"][i, col, rng.integers(R - 5)] = float("inf") if rng.random() < 0.5 else float("-inf")
        for col in range(0, N, 12):
            c["b"][i, col, rng.integers(R - 5)] = float("inf")
    with np.errstate(invalid="ignore"):
        want, err = _want(c)
    assert np.isinf(want).any() and np.isnan(want).any() and np.isfinite(want).any()
    from flashqwen_amd.lora import lora_plan

    plan = lora_plan(_t(c["ids"]), _t(c["cu"]), _meta(c["R"], T), n, T)
    got = _run(c, plan)
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert np.array_equal(np.isinf(g), np.isinf(want))
    assert np.array_equal(g[np.isinf(g)], want[np.isinf(want)])
    fine = np.isfinite(want)
    _check(torch.from_numpy(np.where(fine, g, 0.0)), np.where(fine, want, 0.0), np.where(fine, err, 0.0), f32,
           "finite columns")


def test_no_rows_of_any_strides(gpu):
    """Tensors without rows have no strides to speak of (numpy's come with zeros): nothing is launched."""
    import torch

    from flashqwen_amd.lora import lora_add, lora_plan
    from flashqwen_amd.sample import sample_filtered

    empty = lambda n, dt: torch.empty(0, n, dtype=dt, device=gpu).as_strided((0, n), (0, 0))  # noqa: E731
    i32 = dict(dtype=torch.int32, device=gpu)
    plan = lora_plan(torch.zeros(1, **i32), torch.zeros(2, **i32), _t(np.zeros(16, np.int32)), 2, 0)
    a = torch.zeros(2, 16, 128, dtype=torch.bfloat16, device=gpu)
    b = torch.zeros(2, 64, 16, dtype=torch.bfloat16, device=gpu)
    x, y = empty(128, torch.bfloat16), empty(64, torch.bfloat16)
    for out in (None, y, empty(64, torch.bfloat16)):
        assert lora_add(y, x, a, b, torch.ones(2, device=gpu), plan, out=out).shape == (0, 64)
    v = torch.zeros(0, device=gpu)
    assert sample_filtered(empty(50, torch.float32), v, torch.zeros(0, **i32), v, v, v).shape == (0,)
