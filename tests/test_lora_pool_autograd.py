"""What the adapter pool's autograd wrapper refuses, and what it takes."""
import pytest
import torch

import foundry_attn as fa
from foundry_attn import FoundryAttnError


def test_scales_that_require_a_gradient():
    """Refused before any device work, instead of a gradient that never comes."""
    x, a, b, y = torch.zeros(4, 8), torch.zeros(2, 3, 8), torch.zeros(2, 6, 3), torch.zeros(4, 6)
    plan = fa.LoraPoolPlan(4, 2, torch.zeros(1024, dtype=torch.uint8))
    for scales in (torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True) * 2):
        with pytest.raises(FoundryAttnError, match="scales require a gradient"):
            fa.lora_pool(x.requires_grad_(), a, b, y, scales, plan)


@pytest.mark.gpu
def test_scales_under_no_grad(device):
    """Where nothing is recorded, they are as any others."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x, a, b, y = (torch.randn(*s, generator=g, device="cuda") for s in ((9, 8), (2, 3, 8), (2, 6, 3), (9, 6)))
    plan = fa.lora_pool_plan(torch.arange(9, dtype=torch.int32, device="cuda") % 3, 2)
    scales = torch.tensor([0.5, 2.0], device="cuda")
    want = fa.lora_pool(x, a, b, y, scales, plan)
    with torch.no_grad():
        assert torch.equal(fa.lora_pool(x, a, b, y, scales.clone().requires_grad_(), plan), want)
