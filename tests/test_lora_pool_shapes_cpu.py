"""Operands of the wrong number of dimensions are the pool's own errors, before
anything is allocated for them."""
import pytest
import torch

import foundry_attn as fa
from foundry_attn import FoundryAttnError


@pytest.mark.parametrize("name,shape", [("x", ()), ("x", (8,)), ("x", (2, 4, 8)), ("a", (8,)), ("a", (3, 8)), ("b", (6,)),
                                        ("b", (6, 3)), ("a", ()), ("b", (2, 6, 3, 1))])
def test_dimensions(name, shape):
    t = dict(x=torch.zeros(4, 8), a=torch.zeros(2, 3, 8), b=torch.zeros(2, 6, 3))
    t[name] = torch.zeros(shape)
    plan = fa.LoraPoolPlan(4, 2, torch.zeros(1024, dtype=torch.uint8))
    with pytest.raises(FoundryAttnError):
        fa.lora_pool_fwd(t["x"], t["a"], t["b"], torch.zeros(4, 6), torch.ones(2), plan)
    with pytest.raises(FoundryAttnError):
        fa.lora_pool_bwd(t["x"], t["a"], t["b"], torch.zeros(4, 3), torch.zeros(4, 6), torch.ones(2), plan)
