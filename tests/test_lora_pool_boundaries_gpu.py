"""The adapter pool on both sides of what its launches switch at: a plan that keeps
the index in LDS (up to 8192 tokens and 1024 adapters) or reads it twice, and grids
of more row tiles than one grid axis holds (32768).  Sums of whole numbers under
2^24: every result has to be equal to the exact one."""
import pytest
import torch

from test_lora_pool_gpu import exact, make, run

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def whole_numbers(T, L, K, M, r, dt):
    d = make(T, L, K, M, r, dt, seed=T + L)
    g = torch.Generator(device="cuda").manual_seed(T)
    for k in ("x", "a", "b", "y", "dy", "dx"):
        d[k] = torch.randint(-1, 2, d[k].shape, generator=g, device="cuda").to(dt)
    d["scales"].fill_(1.0)
    return d


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("T,L,K,M,r", [(8191, 5, 8, 8, 2), (8192, 5, 8, 8, 2), (8193, 5, 8, 8, 2), (8192, 1024, 8, 8, 1),
                                       (3000, 1024, 8, 8, 2), (3000, 1025, 8, 8, 2), (2200000, 3, 8, 8, 1)])
def test_equal_to_the_exact_sums(device, T, L, K, M, r, dt):
    d = whole_numbers(T, L, K, M, r, dt)
    got, want = run(d), exact(d)
    for k in got:
        assert torch.equal(got[k].double(), want[k][0]), k
