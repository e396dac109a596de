"""Refusals of the adapters' and the filtered sampler's calls, on the CPU: workspaces that are not one
stretch of memory, widths past what column indexes hold."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from flashqwen_amd import _lib, lora
from flashqwen_amd.sample import sample_filtered

I32 = torch.int32


@pytest.mark.parametrize("workspace", ["expanded", "strided"])
def test_workspaces_of_one_stretch(workspace):
    """A workspace's elements say how many bytes may be written from its first on: an expanded tensor
    has fewer, a strided one has others' among them."""
    ws = torch.empty(1, dtype=torch.uint8).expand(1 << 20) if workspace == "expanded" else \
        torch.empty(1 << 21, dtype=torch.uint8)[::2]
    bf = torch.bfloat16
    plan = lora.LoraPlan(torch.zeros(4, dtype=I32), torch.zeros(2, 4, dtype=I32), torch.zeros(4, dtype=I32))
    y = torch.zeros(4, 128, dtype=bf)
    with pytest.raises(ValueError, match="workspace"):
        lora.lora_add(y, torch.zeros(4, 64, dtype=bf), torch.zeros(2, 16, 64, dtype=bf),
                      torch.zeros(2, 128, 16, dtype=bf), torch.ones(2), plan, out=y, workspace=ws)
    v = torch.zeros(2)
    with pytest.raises(ValueError, match="workspace"):
        sample_filtered(torch.zeros(2, 8), v, torch.zeros(2, dtype=I32), v, v, v, workspace=ws)


def test_widths_past_the_column_indexes():
    """n_out up to 2^30: above it, sums of a column and a workgroup's columns would pass 32 bits."""
    lib = _lib.load()
    buf = C.create_string_buffer(512)
    ptr = (C.addressof(buf) + 255) & ~255  # never read: no such call is launched

    def weights(*ends):
        return _lib.FqaLora(ptr, ptr, ptr, None, 2, 16, 64, len(ends), (C.c_int32 * 4)(*ends))

    for ends in ((2 ** 31 - 64,), (2 ** 30 + 64,), (64, 2 ** 31 - 64), (2 ** 30, 2 ** 30 + 64)):
        w = C.byref(weights(*ends))
        assert lib.fqa_lora_workspace_bytes(w, 4, 2) == _lib.FQA_EUNSUPPORTED, ends
        assert lib.fqa_lora_workspace_most(w, 4) == _lib.FQA_EUNSUPPORTED, ends
        assert lib.fqa_lora_add(w, ptr, 64, ptr, ptr, ptr, 4, 2, ptr, 1 << 31, ptr, 1 << 31, 0, ptr, 1 << 30,
                                None) == _lib.FQA_EUNSUPPORTED, ends
    assert lib.fqa_lora_workspace_bytes(C.byref(weights(2 ** 30)), 4, 2) > 0
