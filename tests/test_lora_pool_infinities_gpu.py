"""Infinities in the adapter pool's inputs: every result is infinite or NaN where
the formulas say so, and what it is without them elsewhere.  The formulas are
evaluated in 64 bits on the host, product by product, for each adapter's tokens."""
import pytest
import torch

import foundry_attn as fa

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def mm(p, q):
    """p q^T by single products, so that a zero or an infinity meets only its own."""
    return (p[:, None, :] * q[None, :, :]).sum(-1)


def formulas(d):
    x, a, b, y, dy, dx, sc = (d[k].double().cpu() for k in ("x", "a", "b", "y", "dy", "dx", "scales"))
    index = d["index"].cpu()
    u, da, db, y, dx = torch.zeros(x.shape[0], a.shape[1]).double(), torch.zeros_like(a), torch.zeros_like(b), y.clone(), dx.clone()
    for i in range(a.shape[0]):
        rows = (index == i).nonzero().flatten()
        if len(rows):
            u[rows], v = mm(x[rows], a[i]), mm(dy[rows], b[i].t())
            y[rows] += sc[i] * mm(u[rows], b[i])
            dx[rows] += sc[i] * mm(v, a[i].t())
            da[i], db[i] = sc[i] * mm(v.t(), x[rows].t()), sc[i] * mm(dy[rows].t(), u[rows].t())
    return dict(u=u, y=y, dx=dx, da=da, db=db)


def run(d):
    plan = fa.lora_pool_plan(d["index"], d["a"].shape[0])
    y, dx = d["y"].clone(), d["dx"].clone()
    u = fa.lora_pool_fwd(d["x"], d["a"], d["b"], y, d["scales"], plan)
    da, db = fa.lora_pool_bwd(d["x"], d["a"], d["b"], u, d["dy"], d["scales"], plan, dx=dx)
    return dict(u=u, y=y, da=da, db=db, dx=dx)


def make(T, L, K, M, r, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device="cuda")).to(dt)
    return dict(index=torch.randint(-1, L, (T,), generator=g, device="cuda").to(torch.int32), x=rn(T, K),
                a=rn(L, r, K, std=K ** -0.5), b=rn(L, M, r, std=0.3), y=rn(T, M), dy=rn(T, M), dx=rn(T, K),
                scales=0.5 + torch.rand(L, generator=g, device="cuda"))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("where", ["x", "dy", "a", "b", "x and dy", "a and b", "rows"])
@pytest.mark.parametrize("size", [(40, 2, 30, 24, 1), (90, 3, 70, 200, 4), (150, 2, 300, 140, 16), (600, 2, 40, 72, 7),
                                  (70, 2, 64, 65, 33), (50, 1, 130, 96, 64)], ids=str)
def test_infinite_where_the_formulas_are(device, size, where, dt):
    d = make(*size, dt, seed=sum(size))
    T, L, K, M, r = size
    clean = run(d)
    t = (d["index"] == L - 1).nonzero().flatten()
    for k in ("x", "dy") if where == "rows" else where.split(" and "):
        z = d[k] = d[k].clone()
        if where == "rows":
            z[t[1]], z[t[2], ::2] = INF, -INF
        elif k in ("x", "dy"):
            z[t[0], 5], z[t[-1], 7] = INF, -INF
        else:
            z[L - 1, 0, -1] = -INF
    got, want = run(d), formulas(d)
    for k in got:
        g, w = got[k].double().cpu(), want[k]
        for name, kind in (("nan", torch.isnan), ("+inf", lambda v: v == INF), ("-inf", lambda v: v == -INF)):
            assert torch.equal(kind(g), kind(w)), (k, name, int((kind(g) != kind(w)).sum()), int(kind(w).sum()))
        assert torch.equal(got[k].cpu()[torch.isfinite(w)], clean[k].cpu()[torch.isfinite(w)]), k


@pytest.mark.parametrize("dt", [BF, F32])
def test_finite_past_the_largest_bf16(device, dt):
    """u and v between the largest bf16 (255 2^120) and the largest f32 stay finite:
    u = v = 255 2^120 + 7 2^117, times 2^-20 exactly 2047 2^97."""
    T, M = 20, 24
    big = torch.zeros(T, M, device="cuda")
    big[:, 0], big[:, 1] = 255 * 2.0 ** 120, 7 * 2.0 ** 117
    big = big.to(dt)
    one = torch.zeros(1, 1, M, device="cuda")
    one[0, 0, :2] = 1
    tiny = torch.full((1, M, 1), 2.0 ** -20, device="cuda")
    plan = fa.lora_pool_plan(torch.zeros(T, dtype=torch.int32, device="cuda"), 1)
    scales, want = torch.ones(1, device="cuda"), torch.full((T, M), 2047 * 2.0 ** 97, device="cuda").to(dt)
    y = torch.zeros(T, M, dtype=dt, device="cuda")
    u = fa.lora_pool_fwd(big, one.to(dt), tiny.to(dt), y, scales, plan)
    assert torch.equal(u, torch.full_like(u, 2047 * 2.0 ** 117)) and torch.equal(y, want)
    dx = torch.zeros(T, M, dtype=dt, device="cuda")
    dy = torch.full((T, M), 2.0 ** -20, device="cuda").to(dt)
    _, db = fa.lora_pool_bwd(big, one.to(dt), tiny.to(dt), u, dy, scales, plan, dx=dx)
    assert torch.equal(db, torch.full_like(db, T * 2047 * 2.0 ** 97))
    # v of big rows, in dx
    fa.lora_pool_bwd(big, tiny.view(1, 1, M).to(dt), one.view(1, M, 1).to(dt), u, big, scales, plan, dx=dx.zero_(),
                     want_factors=False)
    assert torch.equal(dx, want)
