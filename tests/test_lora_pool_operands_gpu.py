"""The f32 operands of the adapter pool's second products, u and v: every bit of
them counts in bf16 too, as in the formulas."""
import pytest
import torch

import foundry_attn as fa

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def pairs(T, P, g):
    """Rows of four columns a pair, (h, m, l, d): bf16 values with h + m + l any
    whole number of up to 19 bits, 0 < |d| <= 8.  Its two low-rank values are
    h + m + l and h + m + l + d."""
    w = torch.randint(-2 ** 18 + 1, 2 ** 18, (T, P), generator=g, device="cuda").float()
    h = w.to(BF).float()
    m = (w - h).to(BF).float()
    d = torch.randint(1, 9, (T, P), generator=g, device="cuda").float()
    d *= torch.randint(0, 2, (T, P), generator=g, device="cuda") * 2 - 1
    return torch.stack((h, m, w - h - m, d), -1).reshape(T, 4 * P), d


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("r", [2, 4, 7, 16, 20, 33, 64])
def test_small_differences_of_large_values(device, dt, r):
    """The low-rank values of a pair cancel up to d.  All sums are of whole numbers
    under 2^24, so that every result has to be equal: those numbers have 19 bits,
    and what is left of the first 16 of them is up to 4, half of the largest d."""
    T, L, M, P = 150, 2, 131, min(r // 2, 4)
    g = torch.Generator(device="cuda").manual_seed(r)
    wide, d = pairs(T, P, g)
    index = torch.randint(-1, L, (T,), generator=g, device="cuda").to(torch.int32)
    low = torch.zeros(r, 4 * P, device="cuda")     # [rank][column of wide]
    out = torch.zeros(M, r, device="cuda")         # [column of the result][rank]
    signs = torch.randint(-1, 2, (M, P), generator=g, device="cuda").float()
    for p in range(P):
        low[2 * p, 4 * p:4 * p + 3] = low[2 * p + 1, 4 * p:4 * p + 4] = 1
        out[:, 2 * p], out[:, 2 * p + 1] = -signs[:, p], signs[:, p]
    old = torch.randint(-4, 5, (T, M), generator=g, device="cuda").float()
    has = (index >= 0)[:, None].float()
    scales = torch.tensor([1.0, 2.0], device="cuda")
    want = (old + has * scales[index.clamp_min(0).long()][:, None] * (d @ signs.t())).to(dt)
    plan = fa.lora_pool_plan(index, L)
    rep = lambda t: t.to(dt).expand(L, *t.shape).contiguous()
    # forward: wide is x, low a, out b
    y = old.to(dt, copy=True)
    u = fa.lora_pool_fwd(wide.to(dt), rep(low), rep(out), y, scales, plan)
    assert torch.equal(u, has * (wide @ low.t()))
    assert torch.equal(y, want)
    # backward: wide is dy, b's columns are low, a's rows out
    dx = old.to(dt, copy=True)
    fa.lora_pool_bwd(torch.zeros(T, M, dtype=dt, device="cuda"), rep(out.t().contiguous()), rep(low.t().contiguous()),
                     torch.zeros(T, r, device="cuda"), wide.to(dt), scales, plan, dx=dx)
    assert torch.equal(dx, want)
