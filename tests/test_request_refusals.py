"""Refusals of the adapters' and the filtered sampler's calls, on the CPU: workspaces that are not one
stretch of memory."""
from __future__ import annotations

import pytest
import torch

from flashqwen_amd import lora
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
