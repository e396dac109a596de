"""lora_add in the forms that real sizes take: items of 128 rows whole to a workgroup, shared by two or by
four, in one pass over their rows and in two; K in several chunks a wave, evenly and not; items of 128 rows
among many of one; and the third bf16 part of an fp32 y.  Against a plain form in 64 bits on the GPU."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_lora import _case, _plan, _run

pytestmark = pytest.mark.gpu


def _want64(c):
    """y + the adapters' products in float64, and what the kernel may be off by before the result is
    rounded: fp32 sums of K (and of R) terms lose at most K 2^-24 of the sum of their magnitudes, h in its
    bf16 parts at most 2^-16 of itself (2^-24 in the three of an fp32 y), the scale and the last addition
    round once more each."""
    import torch

    d = lambda t: t.cuda().double()  # noqa: E731
    y, x, a, b = d(c["y"]), d(c["x"]), c["a"].cuda(), c["b"].cuda()
    K, R = x.shape[1], b.shape[2]
    parts = 2.0 ** -24 if c["y"].dtype is torch.float32 else 2.0 ** -16
    of_row = torch.from_numpy(np.repeat(c["ids"], np.diff(c["cu"]))).cuda()
    out, err = y.clone(), torch.zeros_like(y)
    for g in range(c["adapters"]):
        rows = torch.nonzero(of_row == g)[:, 0]
        if not len(rows):
            continue
        r, sc, c0 = int(c["rank"][g]), float(c["scale"][g]), 0
        for s, cols in enumerate(c["slices"]):
            A, B = d(a[g, s * R:s * R + r]), d(b[g, c0:c0 + cols, :r])
            h, habs = x[rows] @ A.t(), x[rows].abs() @ A.abs().t()
            out[rows, c0:c0 + cols] += sc * (h @ B.t())
            herr = K * 2.0 ** -24 * habs + (parts + (2 * R + 1) * 2.0 ** -24) * h.abs()
            err[rows, c0:c0 + cols] += abs(sc) * (herr @ B.abs().t())
            c0 += cols
    err += 2.0 ** -24 * out.abs() * (of_row >= 0)[:, None]
    return out, err


def _check64(got, c, what):
    import torch

    want, err = _want64(c)
    half = 2.0 ** -24 if c["y"].dtype is torch.float32 else 2.0 ** -8
    allow = (err + half * (want.abs() + err)).clamp(min=1e-300)
    worst = float(((got.double() - want).abs() / allow).max())
    print(f"{what}: worst |diff| / allowance {worst:.3f}", flush=True)
    assert worst <= 1.0, what


# requests' rows, adapters, rank_max, K, slices: what the call takes of them
SHAPES = {
    # column tiles x items: 1024 and more, a workgroup to an item
    "whole items, rank 64": ([2000], 1, 64, 64, (16384,)),
    "whole items, rank 128, two passes over the rows": ([1990, 10], 1, 128, 64, (16384,)),
    "whole items, rank 16": ([1500, 500], 1, 16, 128, (8192, 8192)),
    "whole items, rank 32, uneven": ([130, 1900], 2, 32, 64, (16128, 512)),
    # 512 to 1023: two workgroups to an item
    "halves of items, rank 64": ([1000], 1, 64, 64, (16384,)),
    "halves of items, rank 128": ([999], 1, 128, 192, (16384,)),
    # 4 blocks of ranks at most, many rows: K by chunks of 64 to 8 waves, several a wave
    "K 12288, three chunks a wave": ([300], 1, 64, 12288, (256,)),
    "K 4608, two chunks or one": ([300, 410], 2, 64, 4608, (256,)),
    "K 12288, rank 16, mixed": ([1] * 9 + [400, 90, 20, 333], 3, 16, 12288, (192,)),
    "K not split, three chunks or two": ([33000], 1, 48, 1088, (64,)),
    # more than 4 blocks of ranks: A through LDS
    "tiles of 12 blocks, odd chunks": ([2000, 77], 2, 64, 4160, (512, 128, 128)),
    "tiles in two groups": ([600, 450], 2, 128, 2048, (256, 128, 64)),
    "tiles of 8 blocks, K not split": ([20000, 17000], 2, 128, 192, (128,)),
    # items of 128 rows among many of one, one column tile and several to a workgroup
    "long among short": ([1] * 100 + [128, 100], 101, 32, 256, (256,)),
    "long among short, wide": ([1] * 60 + [128, 40], 61, 128, 128, (24576,)),
}


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("name", SHAPES)
def test_forms_of_real_sizes(gpu, name, f32):
    import torch

    T_of, n, R, K, slices = SHAPES[name]
    print(f"[test_forms_of_real_sizes] {name} f32={f32}", flush=True)
    rng = np.random.default_rng(sum(T_of) + R + K)
    c = _case(rng, T_of, n, R, K, slices, f32, none=0.0)
    c["ids"] = (np.arange(len(T_of)) % n).astype(np.int32)
    c["rank"][-1] = R
    plan = _plan(c)
    y = c["y"].cuda()
    got = _run(c, plan, out=torch.full_like(y, 7.0), y=y)
    _check64(got, c, name)
    _run(c, plan, out=y, y=y)
    assert torch.equal(y, got)
    # small whole numbers: every sum is exact in fp32 (below 2^22, in quarters), h in two parts too
    # (|h| <= 2 K < 2^16), so that the result is the 64-bit one rounded, and no term can be missing
    ints = lambda m, like: torch.from_numpy(  # noqa: E731
        rng.integers(-m, m + 1, tuple(like.shape)).astype(np.float32)).to(like.dtype)
    c.update(x=ints(2, c["x"]), a=ints(1, c["a"]), b=ints(2, c["b"]), y=ints(100, c["y"]),
             scale=torch.from_numpy(rng.choice([1.0, -1.0, 2.0], n).astype(np.float32)))
    y = c["y"].cuda()
    want, _ = _want64(c)
    assert float((want - y.double()).abs().max()) < 2 ** 18
    assert torch.equal(_run(c, plan, out=torch.full_like(y, 7.0), y=y), want.to(y.dtype))


@pytest.mark.parametrize("T_of,R,slices", [([1, 2], 16, (64,)), ([1] * 40, 32, (12288, 12288)),
                                           ([300], 64, (256, 64)), ([260], 128, (128,))])
def test_fp32_keeps_all_bits_of_h(gpu, T_of, R, slices):
    """x A^T of 24 bits, exact in fp32, times one 1 in each row of B onto zeros.  The parts are exact, and
    their halves too; but a part that is shared with the next may end one bit below h's 24, so that each
    of the two sums to which the first two parts are added may round, to half a step: 2 x 2^-24 of h.
    Two bf16 parts, as for a bf16 y, are further off."""
    import torch

    print(f"[test_fp32_keeps_all_bits_of_h] {T_of} R={R} {slices}", flush=True)
    rng = np.random.default_rng(R)
    T, N, S, K = sum(T_of), sum(slices), len(slices), 128
    c = _case(rng, T_of, 1, R, K, slices, True, none=0.0, ranks=np.array([R], np.int32))
    # row j of A takes three of x, of 8 bits each and 2^8 apart: their sum is the three side by side
    x = np.zeros((T, K), np.float32)
    place = rng.permutation(K)[:96].reshape(32, 3)
    for k in range(3):
        x[:, place[:, k]] = rng.integers(128 if k == 0 else 0, 256, (T, 32)) * 2.0 ** -(8 * k)
    a = np.zeros((S * R, K), np.float32)
    which = rng.integers(0, 32, S * R)
    for j in range(S * R):
        a[j, place[which[j]]] = 1.0
    b = np.zeros((N, R), np.float32)
    rank_of = rng.integers(0, R, N)
    b[np.arange(N), rank_of] = 1.0
    t = lambda v: torch.from_numpy(np.ascontiguousarray(v, np.float32))  # noqa: E731
    c.update(x=t(x).bfloat16(), a=t(a[None]).bfloat16(), b=t(b[None]).bfloat16(), y=torch.zeros(T, N),
             scale=torch.ones(1), ids=np.zeros(len(T_of), np.int32))
    slice_of = np.repeat(np.arange(S), slices)
    want = (x.astype(np.float64) @ a.T.astype(np.float64))[:, slice_of * R + rank_of]
    got = _run(c, _plan(c)).double().cpu().numpy()
    off = np.abs(got - want)
    print(f"  worst {(off / want).max() * 2 ** 24:.2f} x 2^-24", flush=True)
    assert (off <= 2 * 2.0 ** -24 * want).all()
    hi = t(want).bfloat16().double().numpy()
    two = hi + t(want - hi).bfloat16().double().numpy()
    assert (np.abs(two - want) > 2 * 2.0 ** -24 * want).mean() > 0.5
