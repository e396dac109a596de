"""fqa_sample_filtered where its masses are longest: tails of small weights under one large one."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_sample_filtered import VOCAB, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [VOCAB, 10_500_001, 1 << 24])
def test_long_tails_of_small_weights(gpu, vocab):
    """One logit holds nearly all of the mass, the others 2^-40 of it each: together 1.4e-7 to 1.5e-5.
    top_p cuts within the tail and the draw falls into it.  The token is within (vocab 2^-47 + 1e-12)
    of the mass of where 64-bit weights and wider sums put the cut and the draw."""
    print(f"[test_long_tails_of_small_weights] {vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    lg = (-40.04 * np.log(2) + rng.choice([0.0, 0.01, 0.3], vocab)).astype(np.float32)
    at = int(rng.integers(vocab // 4, vocab // 2))
    lg[at] = 0.0
    w = np.exp(lg.astype(np.float64))
    tail = float(w.sum() - 1)
    # how far below 1 top_p and u are, in shares of the tail (of what fp32 can say)
    shares = [(0.3, 0.5), (0.5, 0.05), (0.5, 0.4), (0.8, 0.1)]
    below = lambda v: np.float32(1) - np.float32(max(1, round(v * tail * 2 ** 24))) * np.float32(2.0 ** -24)  # noqa: E731
    p = np.array([below(a) for a, _ in shares], np.float32)
    u = np.array([below((1 - a) * b) for a, b in shares], np.float32)
    B = len(shares)
    got = _run(np.broadcast_to(lg, (B, vocab)), np.ones(B, np.float32), np.zeros(B, np.int32), p,
               np.zeros(B, np.float32), u)
    order = np.lexsort((np.arange(vocab), -lg))
    run = np.cumsum(w[order].astype(np.longdouble))
    Z, tol = run[-1], vocab * 2.0 ** -47 + 1e-12
    place = np.empty(vocab, np.int64)
    place[order] = np.arange(vocab)
    for b in range(B):
        cut = int((run < float(p[b]) * Z).sum())  # the last place kept
        t = int(got[b])
        vocab_run = np.cumsum(np.where(place <= cut, w, 0.0).astype(np.longdouble))
        kept = vocab_run[-1]
        lo = (vocab_run[t - 1] if t else 0) - float(u[b]) * kept
        hi = vocab_run[t] - float(u[b]) * kept
        front = run[place[t] - 1] if place[t] else 0  # the mass in front of it in the order
        over = front - float(p[b]) * Z
        print(f"  p 1-{1 - p[b]:.3g} u 1-{1 - u[b]:.3g}: token {t} (the large one: {at}), cut at {cut}, "
              f"draw in ({float(lo):.3g}, {float(hi):.3g}], past the cut {float(over):.3g}, "
              f"border {tol:.3g}", flush=True)
        assert over <= tol * float(Z), b
        # (the cut's border moves the kept mass, and so the draw, by as much again)
        assert lo <= 2 * tol * float(Z) and hi >= -2 * tol * float(Z), b
