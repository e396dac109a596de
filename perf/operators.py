"""What single requests of a shared batch ask for beside the shared work, as cases to measure.

Three operators, at Qwen3-8B's sizes (hidden 4096, q|k|v 4096 + 1024 + 1024, intermediate 12288,
vocabulary 151936) and below:

  plan     a step's rows grouped by their requests' adapters, from the pack's outputs
  lora     low-rank adapters of many requests beside one projection: y + scale (x A^T) B^T
  sample   tokens by temperature, top-k, top-p and min-p from given uniform draws
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

HIDDEN, INTER, VOCAB = 4096, 12288, 151936
TILE = 128  # rows of a plan item
# projection -> (input size, output columns of each slice)
PROJ = {"qkv": (HIDDEN, (4096, 1024, 1024)), "o_proj": (HIDDEN, (HIDDEN,)),
        "gate_up": (HIDDEN, (INTER, INTER)), "down": (INTER, (HIDDEN,)),
        "lm_head": (HIDDEN, (VOCAB,))}


def _lora(**kw):
    """`decodes` requests of one row and `prompts` of plo..phi rows (log-uniform), up to
    `budget` rows in all, over `adapters` adapters of ranks up to `rank`; a share `none` of the
    requests has no adapter.  `sizes` seeds the lengths."""
    case = dict(kind="lora", proj="qkv", decodes=0, prompts=0, plo=2, phi=2, budget=8192,
                adapters=1, rank=16, none=0.0, f32=False, sizes=0)
    assert set(kw) <= set(case) | {"name"}, kw
    case.update(kw)
    return case


def _plan(**kw):
    return {k: v for k, v in _lora(**kw).items() if k not in ("proj", "rank", "f32")} | {"kind": "plan"}


def listed():
    return [
        # four interactive users, each with an adapter of their own: launches and latency count
        _lora(name="lora_o_proj_4", proj="o_proj", decodes=4, adapters=4, rank=16, sizes=1),
        # an ordinary decode step: 16 adapters beside q|k|v, a quarter of the requests without
        _lora(name="lora_qkv_64", proj="qkv", decodes=64, adapters=16, rank=16, none=0.25, sizes=2),
        # a full decode batch over many adapters, the widest projection of a layer
        _lora(name="lora_gate_up_250", proj="gate_up", decodes=250, adapters=64, rank=32, sizes=3),
        # decodes beside prompts of ragged lengths, the longest inner size
        _lora(name="lora_down_700", proj="down", decodes=60, prompts=6, plo=20, phi=400,
              budget=700, adapters=8, rank=64, none=0.1, sizes=4),
        # admission: a full prefill budget of prompts, adapters of a high rank
        _lora(name="lora_qkv_8192", proj="qkv", prompts=24, plo=64, phi=4096, adapters=8, rank=64,
              none=0.1, sizes=5),
        # adapted logits, kept in fp32 for the sampler
        _lora(name="lora_lm_head_32", proj="lm_head", decodes=32, adapters=4, rank=16, f32=True,
              sizes=6),
        # the grouping of an ordinary decode step, and of a full engine with prompts
        _plan(name="plan_64", decodes=64, adapters=16, none=0.25, sizes=7),
        _plan(name="plan_2000", decodes=1990, prompts=10, plo=64, phi=2048, adapters=200, none=0.1,
              sizes=8),
        # one user with a chat model's usual settings
        dict(name="sample_1", kind="sample", rows=1, vocab=VOCAB, pad=0, mix="chat"),
        # an ordinary batch of requests with settings of their own, some of them constrained
        dict(name="sample_64", kind="sample", rows=64, vocab=VOCAB, pad=0, mix="mixed"),
        # a full batch of the same
        dict(name="sample_256", kind="sample", rows=256, vocab=VOCAB, pad=0, mix="mixed"),
        # a full batch of wide nuclei: high temperatures, top-p alone
        dict(name="sample_256_nucleus", kind="sample", rows=256, vocab=VOCAB, pad=0, mix="nucleus"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lora", "lora", "lora", "plan", "sample", "sample"])
    sizes = rng.randrange(1 << 16)
    if kind == "sample":
        return dict(kind="sample", rows=_log(rng, 1, 256), vocab=_log(rng, 900, VOCAB),
                    pad=rng.choice([0, 1, 64]), mix=rng.choice(["chat", "mixed", "mixed", "nucleus"]))
    decodes = _log(rng, 1, 250)
    prompts = rng.choice([0, 0, 0, rng.randint(1, 20)])
    batch = dict(decodes=decodes, prompts=prompts, plo=rng.randint(2, 40), phi=_log(rng, 40, 3000),
                 budget=_log(rng, decodes, 8192), adapters=_log(rng, 1, 64),
                 none=rng.choice([0.0, 0.1, 0.5]), sizes=sizes)
    if kind == "plan":
        more = rng.choice([1, 1, 8])
        return _plan(**{**batch, "decodes": decodes * more, "budget": max(batch["budget"], decodes * more)})
    proj = rng.choice(["qkv", "o_proj", "gate_up", "down", "lm_head"])
    if proj in ("gate_up", "lm_head"):  # wide outputs: fewer rows
        most = 900 if proj == "gate_up" else 64
        batch["decodes"] = min(decodes, most)
        batch["budget"] = min(batch["budget"], most)
    return _lora(proj=proj, rank=rng.choice([16, 16, 32, 48, 64, 128]) if proj != "lm_head" else 16,
                 f32=proj == "lm_head" or rng.random() < 0.2, **batch)


# ---- the batch of a plan or lora case ------------------------------------------------------
def _lengths(case):
    """Rows of each request, decodes and prompts in a mixed order, `budget` in all at most."""
    rng = np.random.default_rng(case["sizes"])
    n = [1] * case["decodes"]
    left = max(0, case["budget"] - len(n))
    for _ in range(case["prompts"]):
        k = min(left, int(round(math.exp(rng.uniform(math.log(case["plo"]), math.log(case["phi"]))))))
        if k < 2:
            break
        n.append(k)
        left -= k
    return np.asarray(n, np.int64)[rng.permutation(len(n))]


def _adapters(case, seed):
    """Adapter of each request (-1: none)."""
    rng = np.random.default_rng(seed)
    n = len(_lengths(case))
    ids = rng.integers(0, case["adapters"], n)
    ids[rng.random(n) < case["none"]] = -1
    return ids


def _ranks(case):
    """Ranks of the adapters: half of them the largest, the others anything below."""
    rng = np.random.default_rng(case["sizes"] + 1)
    n, top = case["adapters"], case["rank"]
    return np.where(rng.random(n) < 0.5, top, rng.integers(1, top + 1, n))


def _item_cap(case):
    n = _lengths(case)
    return int(n.sum()) // TILE + min(len(n), case["adapters"] + 1)


def _of_row(adapter, cu, T):
    """Adapter of each of the step's T rows."""
    at = torch.arange(T, dtype=torch.int32, device=cu.device)
    return adapter.long()[torch.searchsorted(cu[1:], at, right=True)]


def _group(adapter, cu, n_adapters, T, cap):
    """The plan in torch operations: rows by adapter (none last), in tiles of TILE rows."""
    dev = adapter.device
    of_row = _of_row(adapter, cu, T)
    of_row = torch.where((of_row >= 0) & (of_row < n_adapters), of_row, n_adapters)
    rows = torch.sort(of_row, stable=True).indices
    count = torch.zeros(n_adapters + 1, dtype=torch.long, device=dev)
    count.scatter_add_(0, of_row, torch.ones_like(of_row))
    first = torch.cumsum(count, 0) - count
    end = torch.cumsum((count + TILE - 1) // TILE, 0)  # items of the adapters up to each
    at = torch.arange(cap, device=dev)
    who = torch.clamp(torch.searchsorted(end, at, right=True), max=n_adapters)
    k = at - torch.where(who > 0, end[who - 1], 0)
    items = torch.stack([torch.where(who < n_adapters, who, -1), first[who] + k * TILE,
                         torch.clamp(count[who] - k * TILE, max=TILE), torch.zeros_like(at)], 1)
    pad = torch.tensor([-1, 0, 0, 0], device=dev)
    items = torch.where((at < end[-1])[:, None], items, pad)
    meta = torch.stack([end[-1], count.sum(), count[:-1].sum(), end[n_adapters - 1]])
    return rows.int(), items.int(), meta.int()


# ---- inputs --------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, seed, gen, dev)
    lens = _lengths(case)
    T, n = int(lens.sum()), case["adapters"]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)
    adapter = torch.tensor(_adapters(case, seed), dtype=torch.int32, device=dev)
    step_meta = torch.zeros(16, dtype=torch.int32, device=dev)  # what the pack says of the step
    step_meta[0], step_meta[8] = T, len(lens)
    s = dict(case=case, adapter=adapter, cu=cu, step_meta=step_meta, T=T)
    if case["kind"] == "plan":
        return s
    K, cols = PROJ[case["proj"]]
    N, R, S = sum(cols), case["rank"], len(cols)
    rank = torch.tensor(_ranks(case), dtype=torch.int32, device=dev)
    used = torch.arange(R, device=dev) < rank[:, None]  # [n, R]
    normal = lambda *z: torch.randn(*z, generator=gen, device=dev)  # noqa: E731
    a = (normal(n, S, R, K) * K ** -0.5 * used[:, None, :, None]).reshape(n, S * R, K).bfloat16()
    b = (normal(n, N, R) * R ** -0.5 * used[:, None, :]).bfloat16()
    s.update(
        x=normal(T, K).bfloat16(), a=a, b=b, rank=rank,
        scale=0.5 + torch.rand(n, generator=gen, device=dev),
        # what the shared projection left, and the buffer that takes the sum
        y=normal(T, N).to(torch.float32 if case["f32"] else torch.bfloat16),
        plan=_group(adapter, cu, n, T, _item_cap(case)))
    s["out"] = torch.empty_like(s["y"])
    return s


# temperatures, top-k, top-p, min-p of a batch's requests
_KINDS = {
    "chat": [(0.7, 20, 0.8, 0.0), (0.6, 20, 0.95, 0.0), (1.0, 40, 1.0, 0.05)],
    "nucleus": [(1.0, 0, 0.95, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 0.99, 0.0)],
    "mixed": [(0.7, 20, 0.8, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 50, 1.0, 0.0),
              (0.8, 0, 0.95, 0.0), (1.2, 0, 1.0, 0.05), (1.0, 400, 0.9, 0.02), (0.6, 20, 0.95, 0.0)],
}


def _prepare_sample(case, seed, gen, dev):
    B, V = case["rows"], case["vocab"]
    rng = np.random.default_rng(seed)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    pick = np.asarray(_KINDS[case["mix"]])[rng.integers(0, len(_KINDS[case["mix"]]), B)]
    wide = torch.empty(B, V + case["pad"], device=dev)
    # a spread-out body and a few likely tokens ahead of it, as a model's logits have
    wide.normal_(generator=gen).mul_(f32(rng.uniform(1.5, 3.0, B))[:, None])
    head = torch.randint(0, V, (B, min(V, 24)), generator=gen, device=dev)
    wide.scatter_add_(1, head, 9.0 * torch.rand(head.shape, generator=gen, device=dev))
    if case["mix"] == "mixed":  # one request in eight is held to a grammar: most tokens are masked
        held = torch.from_numpy(rng.random(B) < 0.125).to(dev)
        off = torch.rand(wide.shape, generator=gen, device=dev) < 0.99
        off[:, 0] = False
        wide.masked_fill_(off & held[:, None], -math.inf)
    t = pick[:, 0]
    return dict(case=case, logits=wide[:, :V], inv_temp=f32(np.where(t > 0, 1 / np.maximum(t, 1e-3), 0.0)),
                top_k=torch.tensor(pick[:, 1], dtype=torch.int32, device=dev), top_p=f32(pick[:, 2]),
                min_p=f32(pick[:, 3]), u=torch.rand(B, generator=gen, device=dev))


# ---- the operators -------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if kind == "plan":
        n, T, cap = s["case"]["adapters"], s["T"], _item_cap(s["case"])
        if own:
            from flashqwen_amd.lora import lora_plan

            return tuple(lora_plan(s["adapter"], s["cu"], s["step_meta"], n, T, item_cap=cap))
        return _group(s["adapter"], s["cu"], n, T, cap)
    if kind == "lora":
        cols = PROJ[s["case"]["proj"]][1]
        if own:
            from flashqwen_amd.lora import lora_add

            return lora_add(s["y"], s["x"], s["a"], s["b"], s["scale"], s["plan"], slices=cols,
                            rank=s["rank"], out=s["out"])
        return _lora_plain(s, cols)
    if own:
        from flashqwen_amd.sample import sample_filtered

        return sample_filtered(s["logits"], s["inv_temp"], s["top_k"], s["top_p"], s["min_p"], s["u"])
    return _sample_plain(s)


def _lora_plain(s, cols):
    """Every row against every adapter's A, what is not its own adapter's put to zero, then one
    product with all the B side by side."""
    n, R, S = s["a"].shape[0], s["case"]["rank"], len(cols)
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    T = x.shape[0]
    of_row = _of_row(s["adapter"], s["cu"], T)
    ids = torch.arange(n, device=x.device)
    mine = (of_row[:, None] == ids)[:, :, None] & (torch.arange(R, device=x.device) < s["rank"][:, None])
    h = (x @ a.reshape(n * S * R, -1).t()).view(T, n, S, R)
    h = torch.where(mine[:, :, None, :], h * s["scale"][:, None, None], 0.0)  # [T, n, S, R]
    parts = [h[:, :, i].reshape(T, n * R) @ w.permute(0, 2, 1).reshape(n * R, -1)
             for i, w in enumerate(torch.split(b, list(cols), 1))]
    return (s["y"].float() + torch.cat(parts, 1)).to(s["y"].dtype)


def _sample_plain(s):
    """Sorted logits and 64-bit masses, filter by filter."""
    lg = s["logits"]
    B, V = lg.shape
    col = lambda t: s[t].double()[:, None]  # noqa: E731
    lg = torch.where(torch.isnan(lg), -math.inf, lg)
    v, order = torch.sort(lg, dim=1, descending=True, stable=True)
    v = v.double()
    w = torch.exp(torch.where(v == v[:, :1], 0.0, v - v[:, :1]) * col("inv_temp"))
    at = torch.arange(V, device=lg.device)
    k = s["top_k"].long()[:, None]
    keep = (v > -math.inf) & ((at < k) | (k <= 0))
    w = torch.where(keep, w, 0.0)
    mass = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    keep &= (before < col("top_p") * mass[:, -1:]) | (col("top_p") >= 1) | (at == 0)
    keep &= w >= torch.clamp(col("min_p"), max=1.0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run_ = torch.cumsum(kept, 1)
    hit = (kept > 0) & (run_ >= col("u") * run_[:, -1:])
    last = (torch.where(kept > 0, at, -1)).amax(1)
    token = torch.where(hit.any(1), hit.int().argmax(1), last)
    token = torch.where(s["inv_temp"] > 0, token, order[:, 0])
    return torch.where(v[:, 0] > -math.inf, token, -1).int()


# ---- the same in 64 bits, from the definitions ---------------------------------------------
def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers: equal or not
    s = prepare(case, seed)
    if case["kind"] == "lora":
        cols = PROJ[case["proj"]][1]
        ends = np.cumsum(cols)
        cu, ids = s["cu"].tolist(), s["adapter"].tolist()
        y = s["y"].double()
        for g in sorted(set(ids) - {-1}):
            rows = torch.tensor([t for r, i in enumerate(ids) if i == g for t in range(cu[r], cu[r + 1])],
                                device=y.device)
            r = int(s["rank"][g])
            for i, (e, c) in enumerate(zip(ends, cols)):
                a = s["a"][g, i * case["rank"]: i * case["rank"] + r].double()
                b = s["b"][g, e - c:e, :r].double()
                y[rows, e - c:e] += s["scale"][g].double() * ((s["x"][rows].double() @ a.t()) @ b.t())
        return y
    out = []
    lg = s["logits"].cpu().numpy().astype(np.float64)
    for b in range(case["rows"]):
        it, k, p, q, u = (float(s[n][b]) for n in ("inv_temp", "top_k", "top_p", "min_p", "u"))
        order = np.lexsort((np.arange(lg.shape[1]), -lg[b]))
        order = order[np.isfinite(lg[b][order])]
        if it <= 0:
            out.append(int(order[0]))
            continue
        order = order[: int(k)] if k > 0 else order
        w = np.exp((lg[b][order] - lg[b][order[0]]) * it)
        if p < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w)[:-1], p * math.fsum(w), side="left"))
            order, w = order[:n], w[:n]
        order = np.sort(order[w >= q])
        run_ = np.cumsum(np.exp((lg[b][order] - lg[b].max()) * it))
        out.append(int(order[min(np.searchsorted(run_, u * run_[-1], side="left"), len(order) - 1)]))
    return torch.tensor(out, dtype=torch.int32)


def work(case):
    if case["kind"] == "sample":
        B, V = case["rows"], case["vocab"]
        return {"bytes": 4 * B * V + 24 * B, "flops": 4 * B * V}
    lens = _lengths(case)
    T, R = int(lens.sum()), len(lens)
    if case["kind"] == "plan":
        return {"bytes": 4 * (2 * R + 1) + 64 + 4 * T + 16 * _item_cap(case) + 16, "flops": 0}
    K, cols = PROJ[case["proj"]]
    N, S = sum(cols), len(cols)
    ids = _adapters(case, 0)  # the share of rows with an adapter, as any seed has it
    rank = _ranks(case)
    met = np.unique(ids[ids >= 0])
    rows_of = np.bincount(np.where(ids >= 0, ids, case["adapters"]), weights=lens,
                          minlength=case["adapters"] + 1)[:-1]
    rk = float((rows_of * rank).sum())
    size = 4 if case["f32"] else 2
    weights = 2 * int(rank[met].sum()) * (S * K + N)
    return {"bytes": 2 * float(rows_of.sum()) * K + 2 * size * T * N + weights + 8 * T,
            "flops": 2 * rk * (S * K + N)}
