"""The orthogonalised optimiser step against the formulas in 64 bits.

Tolerances, counted before the first run (u = 2^-24):
  momentum  one fma per element: 2 u of |beta m| + |g|.
  update    X = T u / norm: u is one or two f32 roundings of g and m (4 u), T one
            rounding of a 64-bit matrix (u), the product sums at most 64 terms
            (64 u) of |T||u|; what T's own error may be is counted through its
            64-bit oracle, which rounds its Gram matrix in another order: 1e-15
            times the growth a^2 per step, against eigenvalues of at least the
            smallest of interest, stays under 1e-6 of the update for the steps
            tested here.  Together 80 u * (|T| |u|) + 2e-6 of the largest update.
  param     the update's tolerance times lr scale, 3 u of |p| for the two
            products, and one rounding to bf16 (2^-8) or f32.
"""
import math

import pytest
import torch

from foundry_attn import block as fb

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
ABC = fb.MUON_COEFFS


def make(shape, dt, seed=0, low_rank=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    grad, mom = 1e-3 * r(*shape), 1e-3 * r(*shape)
    if low_rank and min(shape[-2:]) > 2:
        grad, mom = (t + 0.1 * r(*shape[:-1], 2) @ r(*shape[:-2], 2, shape[-1]) for t in (grad, mom))
    return (0.05 * r(*shape)).to(dt), grad, mom


def exact(p, g, m, lr, beta, wd, steps, nesterov, eps, coeffs, scale):
    """Products as they are written, matrix by matrix, in 64 bits on the host."""
    p, g, m = (t.double().cpu() for t in (p, g, m))
    a, b, c = coeffs
    m = beta * m + g
    u = g + beta * m if nesterov else m
    rows, cols = u.shape[-2:]
    tall = rows > cols
    x = (u.transpose(-1, -2) if tall else u).contiguous()
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    t_abs = None
    first = x
    for _ in range(steps):
        s = x @ x.transpose(-1, -2)
        x = a * x + (b * s + c * s @ s) @ x
    # |T| |u| bound: T = X pinv(X0); |T| <= the largest gain, so take it as gain * row sums of |X0|
    gain = a ** steps if steps else 1.0
    t_abs = torch.full_like(x, gain) * first.abs().amax(-2, keepdim=True)
    if tall:
        x, t_abs = x.transpose(-1, -2), t_abs.transpose(-1, -2)
    sc = math.sqrt(max(1.0, rows / cols)) if scale is None else scale
    return p * (1 - lr * wd) - lr * sc * x, m, lr * abs(sc) * (80 * U * t_abs + 2e-6 * x.abs().amax())


def step_and_check(items, lr=0.02, beta=0.95, wd=0.01, steps=5, nesterov=True, eps=1e-7, coeffs=ABC, scale=None):
    want = [exact(p, g, m, lr, beta, wd, steps, nesterov, eps, coeffs, scale) for p, g, m in items]
    m_tol = [2 * U * ((beta * m).abs() + g.abs()).double().cpu() + 1e-45 for _, g, m in items]
    fb.muon_step_many(items, lr=lr, beta=beta, weight_decay=wd, steps=steps, nesterov=nesterov, eps=eps,
                      coeffs=coeffs, scale=scale)
    for (p, g, m), (wp, wm, tol), mt in zip(items, want, m_tol):
        assert ((m.double().cpu() - wm).abs() <= mt).all()
        half = 2.0 ** -8 if p.dtype == BF else U
        err = (p.double().cpu() - wp).abs()
        bound = tol + 3 * U * wp.abs() + half * wp.abs() + half * tol
        assert (err <= bound).all(), (tuple(p.shape), (err / bound).max().item())


SHAPES = [(1, 1), (1, 300), (300, 1), (4, 64), (16, 16), (16, 1000), (1000, 16), (17, 17), (7, 515), (515, 7),
          (32, 2048), (2049, 33), (48, 700), (64, 64), (64, 4099), (5001, 64), (63, 130), (3, 16, 520), (5, 333, 12)]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_64_bits(device, shape, dt):
    step_and_check([make(shape, dt, seed=1)])


@pytest.mark.parametrize("low_rank", [False, True])
@pytest.mark.parametrize("kw", [dict(steps=0), dict(steps=1), dict(steps=3, nesterov=False), dict(steps=6),
                                dict(coeffs=(1.5, -0.5, 0.0), steps=10), dict(wd=0.0, beta=0.0), dict(scale=0.3),
                                dict(lr=0.0), dict(eps=1e-2)], ids=str)
def test_options(device, kw, low_rank):
    step_and_check([make((16, 700), F32, seed=2, low_rank=low_rank), make((700, 24), F32, seed=3, low_rank=low_rank)],
                   **kw)


def test_singular_values_near_one(device):
    """lr = -1-like probe: with p = 0, decay 0, lr 1 and scale 1 the step is
    -X, whose singular values the five products bring into (0.65, 1.25) from
    anywhere above 1e-2 of the norm."""
    p, g, m = make((32, 900), F32, seed=5)
    p.zero_(), m.zero_()
    fb.muon_step(p, g, m, lr=1.0, beta=0.0, scale=1.0)
    s = torch.linalg.svdvals(p.double().cpu())
    assert 0.65 < s.min() and s.max() < 1.25


def test_many_in_one_call_are_their_own_calls(device):
    """70 tensors of several ranks and sides (more than a launch holds): the
    same bits as one call each, and twice."""
    shapes = [(16, 300), (300, 16), (40, 90), (4, 4100), (64, 65), (2, 8, 100), (1, 5)] * 10
    items = [make(s, BF, seed=i) for i, s in enumerate(shapes)]
    copies = [[t.clone() for t in it] for it in items]
    fb.muon_step_many(items, weight_decay=0.1)
    for it in copies:
        fb.muon_step(*it, weight_decay=0.1)
    for x, y in zip(items, copies):
        assert torch.equal(x[0], y[0]) and torch.equal(x[2], y[2])


def test_zero_and_poisoned_matrices(device):
    """A zero gradient leaves its matrix but for the decay; NaN, an infinity
    and huge or tiny gradients stay in their own matrix."""
    p, g, m = make((6, 16, 200), F32, seed=7)
    m.zero_()
    g[0] = 0
    g[1, 3, 5] = float("nan")
    g[2, 0, 0] = float("inf")
    g[3] *= 1e30
    g[4] *= 1e-30
    p0 = p.clone()
    q, gg, mm = p.clone(), g.clone(), m.clone()
    fb.muon_step(p, g, m, lr=0.02, weight_decay=0.5, eps=1e-38)
    assert torch.allclose(p[0], p0[0] * (1 - 0.01), rtol=3 * U, atol=0)
    assert p[1].isnan().all() and p[2].isnan().all()
    assert torch.isfinite(p[3:]).all()
    for k in (3, 4, 5):
        s = torch.linalg.svdvals(((p0[k].double() * 0.99 - p[k].double()) / 0.02).cpu())
        assert 0.6 < s.min() and s.max() < 1.3, k
    alone = [t[5:6].clone() for t in (q, gg, mm)]
    fb.muon_step(*alone, lr=0.02, weight_decay=0.5, eps=1e-38)
    assert torch.equal(alone[0][0], p[5])


def test_rank_deficient(device):
    """Rows of zeros (a pool's padding up to its rank) stay zero rows, and the
    others get the step of the matrix without them."""
    p, g, m = make((16, 600), F32, seed=8)
    for t in (p, g, m):
        t[10:] = 0
    small = [t[:10].clone() for t in (p, g, m)]
    fb.muon_step(p, g, m, scale=1.0)
    fb.muon_step(*small, scale=1.0)
    assert not p[10:].any() and not m[10:].any()
    assert torch.equal(p[:10], small[0])


def test_stream_and_graph(device):
    """On another stream, and captured: every replay steps the parameters as an
    eager call does."""
    items = [make((16, 3000), BF, seed=1), make((900, 16), BF, seed=2)]
    twin = [[t.clone() for t in it] for it in items]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fb.muon_step_many(items)
    torch.cuda.current_stream().wait_stream(side)
    fb.muon_step_many(twin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fb.muon_step_many(items)
    for k in range(4):
        for it, tw in zip(items, twin):
            it[1].mul_(-1.1)
            tw[1].mul_(-1.1)
        graph.replay()
        fb.muon_step_many(twin)
        torch.cuda.synchronize()
        for it, tw in zip(items, twin):
            assert torch.equal(it[0], tw[0]) and torch.equal(it[2], tw[2]), k


def test_empty_list_and_no_matrices(device):
    fb.muon_step_many([])
    e = torch.empty(0, 4, 8, device="cuda")
    fb.muon_step(e, e.clone(), e.clone())


def test_zero_matrix_under_the_smallest_eps(device):
    """1 / eps^2 leaves the range of f64; the update is still zero."""
    for shape in ((16, 40), (40, 20)):
        p, g, m = make(shape, F32, seed=4)
        g.zero_(), m.zero_()
        before = p.clone()
        fb.muon_step(p, g, m, eps=1e-300)
        assert torch.equal(p, before) and not m.any()


def test_the_same_tensor_twice_is_refused(device):
    p, g, m = make((8, 40), F32)
    other = make((8, 40), F32, seed=1)
    for items in ([(p, g, m), (p, g, other[2])], [(p, g, m), (other[0], g, m)], [(p, g, m)] * 2):
        with pytest.raises(fb.FoundryAttnError):
            fb.muon_step_many(items)
