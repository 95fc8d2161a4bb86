"""Layer norm with weight and bias, forward and backward, against the formulas
in 64 bits.

Tolerances, counted before the first run (u = 2^-24, one f32 rounding):
  mean      sums of C terms in a tree of depth <= 8 (a lane's chunk) * CH + 10
            (the wave and the group): (40 + 3) u of sum|x|/C.
  rstd      the variance the same way, and (x - mean) carries mean's error;
            1e-5 relative covers C <= 32768 at |mean| <= 4 sigma.
  y, dx     f32 arithmetic to 2e-5 of the row's largest term, then one rounding
            to the storage type (bf16 2^-8, f32 2^-24 relative).
  dw, db    sums over N rows in a fixed tree: at most ceil(N / 512) + 40 terms
            in a row: (N / 512 + 60) u of the sum of absolute terms, and n's own
            error (2e-5).
"""
import pytest
import torch

from foundry_attn import block as fb

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}
U = 2.0 ** -24


def make(n, c, dt, wdt, seed=0, offset=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = ((r(n, c) + offset) * torch.exp(0.5 * r(n, 1))).to(dt)
    return x, (1 + 0.2 * r(c)).to(wdt), (0.2 * r(c)).to(wdt), r(n, c).to(dt), r(n, c).to(dt)


def exact(x, w, b, dy, dres, eps):
    x, w, dy = x.double(), w.double(), dy.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    n = (x - mean) * rstd
    y = n * w + (0 if b is None else b.double())
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
    return y, mean[:, 0], rstd[:, 0], dx, (dy * n).sum(0), dy.sum(0), n


def check(got, want, tol, label):
    err = (got.double() - want).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, (label, worst)


def run(x, w, b, dy, dres, eps=1e-5, out=None, dx_out=None):
    y, mean, rstd = fb.layer_norm_fwd(x, w, b, eps, out=out)
    want = exact(x, w, b, dy, dres, eps)
    half = HALF[x.dtype]
    top = lambda t: t.abs().amax(1, keepdim=True)
    check(mean, want[1], 43 * U * x.double().abs().mean(1) + 1e-30, "mean")
    check(rstd, want[2], 1e-5 * want[2], "rstd")
    check(y, want[0], half * want[0].abs() + 2e-5 * (top(want[6]) * w.double().abs().max() + 1), "y")
    dx, dw, db = fb.layer_norm_bwd(x, dy, w, mean, rstd, dres=dres, out=dx_out)
    g = dy.double() * w.double()
    scale = want[2][:, None] * (top(g) + top(want[6]) * top(g))
    if dres is not None:
        scale = scale + top(dres.double())
    check(dx, want[3], half * want[3].abs() + 2e-5 * scale, "dx")
    terms = (x.shape[0] / 512 + 60) * U
    check(dw, want[4], (terms + 2e-5) * (dy.double() * want[6]).abs().sum(0) + 2e-5 * dy.double().abs().sum(0) + 1e-30,
          "dw")
    check(db, want[5], terms * dy.double().abs().sum(0) + 1e-30, "db")
    return y, dx, dw, db


@pytest.mark.parametrize("dt,wdt", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 7), (1, 512), (5, 513), (33, 768), (600, 1001), (17, 1536), (9, 4100),
                                 (3, 8192), (4, 8193), (2, 16390), (2, 32768)])
def test_against_64_bits(device, n, c, dt, wdt):
    x, w, b, dy, dres = make(n, c, dt, wdt)
    run(x, w, b, dy, None)
    run(x, w, None, dy, dres)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("n,c", [(20000, 64), (7001, 640), (3000, 2047)])
def test_many_rows(device, n, c, dt):
    x, w, b, dy, _ = make(n, c, dt, dt, seed=3)
    first = run(x, w, b, dy, None)
    for a, z in zip(first, run(x, w, b, dy, None)):
        assert torch.equal(a, z)


@pytest.mark.parametrize("dt", [BF, F32])
def test_row_strides_and_aliases(device, dt):
    """Column slices at odd offsets; y over x and dx over dy; what lies beside
    the views stays."""
    n, c = 37, 773
    x, w, b, dy, dres = make(n, c, dt, dt, seed=5)
    want = run(x, w, b, dy, dres)
    wide = lambda t, off: torch.full((n, c + 20), 7.0, dtype=dt, device="cuda")[:, off:off + c].copy_(t)
    xs, dys, rs = wide(x, 3), wide(dy, 1), wide(dres, 5)
    ys, dxs = wide(torch.zeros_like(x), 9), wide(torch.zeros_like(x), 7)
    got = run(xs, w, b, dys, rs, out=ys, dx_out=dxs)
    for a, z in zip(got, want):
        assert torch.equal(a, z)
    for t, off in ((ys, 9), (dxs, 7)):
        base = t._base
        assert (base[:, :off] == 7).all() and (base[:, off + c:] == 7).all()
    y, mean, rstd = fb.layer_norm_fwd(xs, w, b)
    fb.layer_norm_bwd(xs, dys, w, mean, rstd, dres=rs, out=dys)
    assert torch.equal(dys, want[1])
    fb.layer_norm_fwd(xs, w, b, out=xs)
    assert torch.equal(xs, want[0])


def test_no_rows(device):
    x = torch.empty(0, 40, dtype=BF, device="cuda")
    w = torch.ones(40, device="cuda")
    y, mean, rstd = fb.layer_norm_fwd(x, w, w)
    dx, dw, db = fb.layer_norm_bwd(x, x, w, mean, rstd)
    assert y.shape == dx.shape == (0, 40) and not dw.any() and not db.any()


def test_rows_apart(device):
    """A row of NaN, one of infinities and a constant one leave the others'
    results as they are."""
    x, w, b, dy, _ = make(40, 600, F32, F32, seed=9)
    y0, mean, rstd = fb.layer_norm_fwd(x, w, b)
    dx0 = fb.layer_norm_bwd(x, dy, w, mean, rstd)[0]
    z = x.clone()
    z[7], z[20, 3], z[30] = float("nan"), float("inf"), 2.5
    y, mean, rstd = fb.layer_norm_fwd(z, w, b)
    dx = fb.layer_norm_bwd(z, dy, w, mean, rstd)[0]
    keep = [i for i in range(40) if i not in (7, 20, 30)]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(dx[keep], dx0[keep])
    assert y[7].isnan().all() and y[20].isnan().any()
    assert torch.allclose(y[30], b, atol=1e-3) and torch.isfinite(dx[30]).all()


def test_only_what_is_wanted(device):
    x, w, b, dy, _ = make(50, 300, BF, F32, seed=2)
    y, mean, rstd = fb.layer_norm_fwd(x, w, b)
    dx, dw, db = fb.layer_norm_bwd(x, dy, w, mean, rstd)
    a = fb.layer_norm_bwd(x, dy, w, mean, rstd, want_dweight=False)
    c = fb.layer_norm_bwd(x, dy, w, mean, rstd, want_dbias=False)
    d = fb.layer_norm_bwd(x, dy, w, mean, rstd, want_dweight=False, want_dbias=False)
    assert a[1] is None and c[2] is None and d[1] is None and d[2] is None
    assert torch.equal(a[2], db) and torch.equal(c[1], dw)
    assert all(torch.equal(t[0], dx) for t in (a, c, d))


def test_autograd_matches_differences(device):
    """The wrapper's gradients against central differences in 64 bits of the
    same formula (h = 1e-4: truncation h^2, cancellation 1e-16 / h)."""
    x, w, b, dy, _ = make(6, 50, F32, F32, seed=4)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = fb.layer_norm(x.view(2, 3, 50), w, b)
    y.backward(dy.view(2, 3, 50))
    loss = lambda xx, ww, bb: (exact(xx, ww, bb, dy, None, 1e-5)[0] * dy.double()).sum().item()
    h = 1e-4
    for t, k in ((x, 0), (w, 1), (b, 2)):
        for at in ((0,) if t.dim() == 1 else (0, 3), (17,) if t.dim() == 1 else (5, 49)):
            args = [x.detach().double(), w.detach().double(), b.detach().double()]
            lo, hi = list(args), list(args)
            lo[k], hi[k] = args[k].clone(), args[k].clone()
            lo[k][at] -= h
            hi[k][at] += h
            want = (loss(*hi) - loss(*lo)) / (2 * h)
            assert abs(t.grad[at].item() - want) < 1e-4 * (1 + abs(want)), (k, at)


@pytest.mark.parametrize("layout", ["expanded", "transposed"])
def test_autograd_of_inputs_without_rows(device, layout):
    """A broadcast or transposed x and upstream gradient: what a copy gives."""
    x0, w0, b0, dy, _ = make(20, 20, F32, F32, seed=6)
    view = (lambda t: t[:1].expand(20, 20)) if layout == "expanded" else (lambda t: t.t())
    got = []
    for lay in (view, lambda t: view(t).contiguous()):
        x, w, b = (t.clone().requires_grad_() for t in (x0, w0, b0))
        y = fb.layer_norm(lay(x), w, b)
        y.backward(lay(dy))
        got.append([y, x.grad, w.grad, b.grad])
    assert all(torch.equal(p, q) for p, q in zip(*got)) and got[0][1].any()


def test_other_stream_and_graph(device):
    x, w, b, dy, _ = make(300, 1030, BF, BF, seed=6)
    want = run(x, w, b, dy, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, dy, None)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, z) for a, z in zip(got, want))

    def step():
        y, mean, rstd = fb.layer_norm_fwd(x, w, b)
        return (y, *fb.layer_norm_bwd(x, dy, w, mean, rstd))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        x.mul_(-1.25)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, z) for a, z in zip(outs, step())), k
