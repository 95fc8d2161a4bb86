"""Where a NaN or an infinity of a gradient shows in the orthogonalised step."""
import pytest
import torch

from foundry_attn import block as fb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(8, 40), (300, 16), (24, 600), (64, 70)])
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_reach(device, shape, steps, value):
    g = torch.Generator(device="cuda").manual_seed(1)
    p, grad = torch.randn(*shape, generator=g, device="cuda"), torch.randn(*shape, generator=g, device="cuda")
    at = (3, 7)
    grad[at] = value
    fb.muon_step(p, grad, torch.zeros_like(p), steps=steps)
    want = torch.ones(shape, dtype=torch.bool, device="cuda")
    if steps == 0 and value == value:
        want.zero_()
        want[(slice(None), at[1]) if shape[0] <= shape[1] else (at[0], slice(None))] = True
    assert torch.equal(p.isnan(), want)
    assert torch.isfinite(p[~want]).all()
