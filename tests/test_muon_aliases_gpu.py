"""A gradient of the orthogonalised step that is also one of its params or momenta
would be overwritten between the step's two readings of it."""
import pytest
import torch

from foundry_attn import FoundryAttnError
from foundry_attn import block as fb

pytestmark = pytest.mark.gpu


def make(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(8, 40, generator=g, device="cuda") for _ in range(3)]


def test_gradients_among_what_is_written(device):
    p, g, m = make(0)
    q, h, n = make(1)
    for items in ([(p, m, m)], [(p, p, m)], [(p, n, m), (q, h, n)], [(p, g, m), (q, p, n)]):
        before = [t.clone() for it in items for t in it]
        with pytest.raises(FoundryAttnError, match="gradient"):
            fb.muon_step_many(items)
        assert all(torch.equal(a, b) for a, b in zip(before, [t for it in items for t in it]))


def test_items_may_share_a_gradient(device):
    p, g, m = make(2)
    q, _, n = make(3)
    want = [t.clone() for t in (p, m, q, n)]
    fb.muon_step(want[0], g, want[1])
    fb.muon_step(want[2], g, want[3])
    fb.muon_step_many([(p, g, m), (q, g, n)])
    assert all(torch.equal(a, b) for a, b in zip((p, m, q, n), want))
