"""Token sampling on the GPU through the C ABI (fqa_sample; LaunchSampleBatch,
engine/src/kernels.cu:184-327): greedy rows (inv_temp <= 0) and temperature + top-p rows
with the caller's uniform draws, torch tensors as device memory."""
from __future__ import annotations

import torch

from ._launch import launch
from ._lib import check, load


def _ptr(t: torch.Tensor):
    return t.data_ptr()


def sample(logits: torch.Tensor, inv_temp: torch.Tensor, top_p: torch.Tensor,
           u: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """logits [B, N] fp32 (rows may be strided), inv_temp / top_p / u [B] fp32 -> [B] int32
    tokens, on the current stream."""
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be a 2-D fp32 tensor with unit column stride")
    B, N = logits.shape
    for name, t in (("inv_temp", inv_temp), ("top_p", top_p), ("u", u)):
        if t.dtype != torch.float32 or t.shape != (B,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous fp32 tensor of shape ({B},)")
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    stream = torch.cuda.current_stream(logits.device).cuda_stream
    check(load().fqa_sample(_ptr(logits), B, N, logits.stride(0), _ptr(inv_temp), _ptr(top_p),
                            _ptr(u), _ptr(out), stream), "fqa_sample")
    return out


def sample_filtered(logits: torch.Tensor, inv_temp: torch.Tensor, top_k: torch.Tensor,
                    top_p: torch.Tensor, min_p: torch.Tensor, u: torch.Tensor,
                    out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Tokens by temperature, top-k, top-p and min-p (fqa_sample_filtered): logits [B, N] fp32 (rows
    may be strided), inv_temp / top_p / min_p / u [B] fp32, top_k [B] int32 -> [B] int32 tokens, on
    the current stream of the logits' device; -1 for a row with nothing to pick."""
    if logits.dtype != torch.float32 or logits.dim() != 2 or (logits.stride(1) != 1 and logits.numel() > 0):
        raise ValueError("logits must be a 2-D fp32 tensor with unit column stride")
    index = logits.get_device()
    B, N = logits.shape
    for name, t in (("inv_temp", inv_temp), ("top_p", top_p), ("min_p", min_p), ("u", u)):
        _check_row_values(name, t, torch.float32, B, index)
    _check_row_values("top_k", top_k, torch.int32, B, index)
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    else:
        _check_row_values("out", out, torch.int32, B, index)
    if workspace is None:
        need = load().fqa_sample_filtered_workspace_bytes(B, N)
        if need < 0:
            check(need, "fqa_sample_filtered_workspace_bytes")
        workspace = torch.empty(need or 16, dtype=torch.uint8, device=logits.device)
    elif workspace.get_device() != index or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {logits.device}")
    launch(index, "fqa_sample_filtered", logits.data_ptr(), B, N, logits.stride(0) if B > 1 else N,
           inv_temp.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), min_p.data_ptr(), u.data_ptr(),
           out.data_ptr(), workspace.data_ptr(), workspace.nbytes)
    return out


def _check_row_values(name: str, t: torch.Tensor, dtype: torch.dtype, n: int, index: int) -> None:
    if t.dtype is not dtype or t.dim() != 1 or t.size(0) != n or not t.is_contiguous() \
            or t.get_device() != index:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape ({n},) on the logits' device")
