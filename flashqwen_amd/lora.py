"""Low-rank adapters of many requests beside a shared projection, through the C ABI
(fqa_lora_plan, fqa_lora_add), torch tensors as device memory: y + scale (x A^T) B^T with each
row's own adapter."""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Sequence

import torch

from . import _lib
from ._launch import launch
from ._lib import FqaLora, check, load

TILE_ROWS = _lib.FQA_LORA_TILE_ROWS


class LoraPlan(NamedTuple):
    """A step's rows grouped by adapter (fqa_lora_plan)."""

    rows: torch.Tensor  # [rows_bound] int32, the step's rows in the plan's order
    items: torch.Tensor  # [item_cap, 4] int32 {adapter or -1, first, count, 0}
    meta: torch.Tensor  # [4] int32 items, rows, adapted rows, adapted items


class LoraWeights(NamedTuple):
    """The adapters of one projection, laid out as lora_add takes them."""

    a: torch.Tensor  # [n, slices * rank_max, n_in] bf16
    b: torch.Tensor  # [n, n_out, rank_max] bf16
    scale: torch.Tensor  # [n] fp32
    rank: torch.Tensor  # [n] int32
    slices: tuple[int, ...]  # output columns of each slice


def item_bound(n_reqs: int, rows: int, n_adapters: int) -> int:
    """The most items a plan of these bounds can have."""
    return int(load().fqa_lora_item_bound(n_reqs, rows, n_adapters))


def _int32(name: str, t: torch.Tensor, index: int, n: int = 0) -> None:
    if t.dtype is not torch.int32 or not t.is_contiguous() or t.numel() < n or t.get_device() != index:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements or more on the "
                         "device of the others")


def _check_plan(rows, items, meta, index: int) -> None:
    i32 = torch.int32
    if not (rows.dtype is i32 and items.dtype is i32 and meta.dtype is i32 and rows.dim() == 1
            and items.dim() == 2 and items.size(1) == 4 and meta.numel() >= _lib.FQA_LORA_META_LEN
            and rows.is_contiguous() and items.is_contiguous() and meta.is_contiguous()
            and rows.get_device() == items.get_device() == meta.get_device() == index):
        raise ValueError("a plan is contiguous int32 tensors rows [rows], items [items, 4] and meta [4] on "
                         "the device of the others")


def lora_plan(adapter: torch.Tensor, cu_seqlens: torch.Tensor, meta: torch.Tensor,
              n_adapters: int, rows_bound: int, *, n_reqs: int | None = None,
              req_map: torch.Tensor | None = None, item_cap: int | None = None,
              out: LoraPlan | None = None) -> LoraPlan:
    """Group a packed step's rows by adapter, on the current stream.  adapter [ids] int32: each
    request's adapter, anything outside [0, n_adapters) for none; cu_seqlens and meta are the
    pack's (AttnStep.cu_seqlens, .meta).  req_map: the batch's index into `adapter` per request
    (AttnStep.sel_req after schedule_and_prepare).  n_reqs bounds the requests (default: what
    `adapter` or `req_map` holds), rows_bound the rows.  `out` (an earlier plan of these bounds)
    is written in place of new tensors."""
    index = adapter.get_device()
    ids = adapter.numel()
    if n_reqs is None:
        n_reqs = ids if req_map is None else req_map.numel()
    _int32("adapter", adapter, index, n_reqs if req_map is None else 0)
    if req_map is not None:
        _int32("req_map", req_map, index, n_reqs)
    _int32("cu_seqlens", cu_seqlens, index, n_reqs + 1)
    _int32("meta", meta, index, _lib.META_LEN)
    if item_cap is None:
        item_cap = item_bound(n_reqs, rows_bound, n_adapters) if out is None else out[1].size(0)
    if out is None:
        i32 = dict(dtype=torch.int32, device=adapter.device)
        out = LoraPlan(torch.empty(max(rows_bound, 0), **i32), torch.empty(max(item_cap, 0), 4, **i32),
                       torch.empty(_lib.FQA_LORA_META_LEN, **i32))
    else:
        _check_plan(*out, index)
        if out[0].numel() < rows_bound or out[1].size(0) < item_cap:
            raise ValueError("out is smaller than the plan's bounds")
    launch(index, "fqa_lora_plan", adapter.data_ptr(), ids,
           req_map.data_ptr() if req_map is not None else None, cu_seqlens.data_ptr(),
           meta.data_ptr(), n_reqs, rows_bound, n_adapters, out[0].data_ptr(), out[1].data_ptr(),
           item_cap, out[2].data_ptr())
    return out


def lora_weights(adapters: Sequence, slices: Sequence[int], device="cuda") -> LoraWeights:
    """Lay out adapters for lora_add.  Each is (a, b, scale): a the [rank, n_in] matrices and b the
    [columns, rank] matrices of the projection's slices (or one of each where there is one slice),
    all of one rank; ranks may differ between adapters."""
    slices = tuple(int(c) for c in slices)
    one = lambda m: [m] if isinstance(m, torch.Tensor) else list(m)  # noqa: E731
    adapters = [(one(a), one(b), float(scale)) for a, b, scale in adapters]
    if not adapters:
        raise ValueError("no adapters")
    n_in = adapters[0][0][0].shape[1]
    for a, b, _ in adapters:
        r = a[0].shape[0]
        if len(a) != len(slices) or len(b) != len(slices) or any(
                m.shape != (r, n_in) for m in a) or any(
                m.shape != (c, r) for m, c in zip(b, slices)):
            raise ValueError("an adapter's matrices are not [rank, n_in] and [columns, rank] per slice")
    top = max(a[0].shape[0] for a, _, _ in adapters)
    R = max(16, -(-top // 16) * 16)
    n, S = len(adapters), len(slices)
    wa = torch.zeros(n, S, R, n_in, dtype=torch.bfloat16, device=device)
    wb = torch.zeros(n, sum(slices), R, dtype=torch.bfloat16, device=device)
    for i, (a, b, _) in enumerate(adapters):
        r = a[0].shape[0]
        for s, m in enumerate(a):
            wa[i, s, :r] = m.to(wa)
        wb[i, :, :r] = torch.cat([m.to(wb) for m in b])
    return LoraWeights(
        wa.view(n, S * R, n_in), wb,
        torch.tensor([s for _, _, s in adapters], dtype=torch.float32, device=device),
        torch.tensor([a[0].shape[0] for a, _, _ in adapters], dtype=torch.int32, device=device),
        slices)


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
             scale: torch.Tensor, plan: LoraPlan, slices: Sequence[int] | None = None,
             rank: torch.Tensor | None = None, out: torch.Tensor | None = None,
             workspace: torch.Tensor | None = None) -> torch.Tensor:
    """out = y + the adapters' products, row by row of the plan, on the current stream: y [rows,
    n_out] bf16 or fp32 (what the projection left), x [rows, n_in] bf16 (row strides allowed), a
    [n, slices * rank_max, n_in] and b [n, n_out, rank_max] bf16, scale [n] fp32, rank [n] int32
    (default: rank_max for all).  `out` may be y (in place, rows without an adapter untouched).
    Rows that the plan does not hold, and rows of adapters that a and b do not have, are left as
    they were in `out`; without it a new tensor is returned, a copy of y that the products are
    added to, so these rows are y's there (the copy is a pass of its own over y)."""
    index = x.get_device()
    bf16 = torch.bfloat16
    f32 = y.dtype is torch.float32
    if x.dtype is not bf16 or a.dtype is not bf16 or b.dtype is not bf16:
        raise ValueError("x, a and b must be bf16")
    if not f32 and y.dtype is not bf16:
        raise ValueError("y must be bf16 or fp32")
    T, K = x.shape
    rows_y, N = y.shape
    n, SR, Ka = a.shape
    nb, Nb, R = b.shape
    ldx, cx = x.stride()
    ldy, cy = y.stride()
    if rows_y != T or (T > 0 and (cx != 1 or cy != 1)):
        raise ValueError("x and y must have unit column stride and the same rows")
    slices = (N,) if slices is None else tuple(slices)
    S, total, ends = _ends(slices)
    if total != N:
        raise ValueError(f"slices {slices} do not make up {N} columns")
    if Ka != K or SR != S * R or nb != n or Nb != N or not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit x, y and the slices, or "
                         "are not contiguous")
    if scale.dtype is not torch.float32 or scale.numel() != n or not scale.is_contiguous():
        raise ValueError(f"scale must be a contiguous fp32 tensor of {n} elements")
    if rank is not None:
        _int32("rank", rank, index, n)
    rows, items, meta = plan
    _check_plan(rows, items, meta, index)
    rows_bound, item_bound_ = rows.numel(), items.size(0)
    if rows_bound > T:
        raise ValueError(f"the plan holds up to {rows_bound} rows, x has {T}")
    if T == 1:  # the row stride of a single row may be anything
        ldx, ldy = K, N
    if out is None:
        y = out = y.detach().clone(memory_format=torch.contiguous_format)
        ldy = ldo = N
    elif out is y:
        ldo = ldy
    else:
        ldo, co = out.stride()
        if out.dtype is not y.dtype or (co != 1 and T > 0) or out.size(0) != T or out.size(1) != N:
            raise ValueError("out must have y's dtype and shape and unit column stride")
        if T == 1:
            ldo = N
    if not (index == y.get_device() == a.get_device() == b.get_device() == scale.get_device()
            == out.get_device()):
        raise ValueError("all tensors must be on one device")
    w = FqaLora(a.data_ptr(), b.data_ptr(), scale.data_ptr(),
                rank.data_ptr() if rank is not None else None, n, R, K, S, ends)
    w_ref = C.byref(w)
    if workspace is None:
        nbytes = load().fqa_lora_workspace_bytes(w_ref, rows_bound, item_bound_)
        if nbytes < 0:
            check(nbytes, "fqa_lora_workspace_bytes")
        nbytes = nbytes or 16
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    else:
        nbytes = workspace.nbytes
        if workspace.get_device() != index or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on {x.device}")
    launch(index, "fqa_lora_add", w_ref, x.data_ptr(), ldx, rows.data_ptr(), items.data_ptr(),
           meta.data_ptr(), rows_bound, item_bound_, y.data_ptr(), ldy, out.data_ptr(), ldo, f32,
           workspace.data_ptr(), nbytes)
    return out


@functools.lru_cache(maxsize=64)
def _ends(slices: tuple[int, ...]):
    if not 1 <= len(slices) <= _lib.FQA_LORA_MAX_SLICES:
        raise ValueError(f"{len(slices)} slices: 1 to {_lib.FQA_LORA_MAX_SLICES} are supported")
    ends = [sum(slices[: i + 1]) for i in range(len(slices))]
    return len(slices), ends[-1], (C.c_int32 * _lib.FQA_LORA_MAX_SLICES)(*ends)
