"""The pool of adapters against the formulas in 64 bits, adapter by adapter.

Tolerances, counted before the first run (u = 2^-24, every sum below of absolute
terms of the exact values):
  u, v   K (or M) products in f32: at most K / 4 + 64 roundings in a row.
  y, dx  the term's operand as two bf16 parts (2^-16 of it left at most), 64 + 64
         roundings over the rank, the error of u or v carried through |B| or |A|,
         then one rounding of the result to the storage type (bf16 2^-8, f32 u).
  da, db T_i products in f32 (T_i + 64 roundings), the operand in three parts
         (2^-23), and the error of v or u carried through.
"""
import pytest
import torch

import foundry_attn as fa

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
HALF = {BF: 2.0 ** -8, F32: U}


def make(T, L, K, M, r, dt, index=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device="cuda")).to(dt)
    if index is None:
        index = torch.randint(-1, L, (T,), generator=g, device="cuda").to(torch.int32)
    return dict(index=index, x=rn(T, K), a=rn(L, r, K, std=K ** -0.5), b=rn(L, M, r, std=0.3), y=rn(T, M),
                scales=0.5 + torch.rand(L, generator=g, device="cuda"), dy=rn(T, M), dx=rn(T, K))


def exact(d):
    """Results and their tolerances."""
    x, a, b, y, dy, dx, sc = (d[k].double() for k in ("x", "a", "b", "y", "dy", "dx", "scales"))
    T, K = x.shape
    L, r = a.shape[:2]
    M = b.shape[1]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")
    u, ue, ye, da, dae, db, dbe, dxe = (z(T, r), z(T, r), z(T, M), z(L, r, K), z(L, r, K), z(L, M, r), z(L, M, r),
                                        z(T, K))
    y, dx = y.clone(), dx.clone()
    two = 2.0 ** -16 if d["x"].dtype == BF else 0.0
    mm = lambda p, q: torch.mm(p.contiguous(), q.contiguous())
    for i in range(L):
        rows = (d["index"] == i).nonzero().flatten()
        if not len(rows):
            continue
        s, n = sc[i], len(rows)
        xi, dyi, A, B = x[rows], dy[rows], a[i], b[i]
        ui, vi = mm(xi, A.t()), mm(dyi, B)
        uei = (K / 4 + 64) * U * mm(xi.abs(), A.abs().t())
        vei = (M / 4 + 64) * U * mm(dyi.abs(), B.abs())
        u[rows], ue[rows] = ui, uei
        y[rows] += s * mm(ui, B.t())
        ye[rows] = s * mm(uei + (two + 130 * U) * ui.abs(), B.abs().t())
        dx[rows] += s * mm(vi, A)
        dxe[rows] = s * mm(vei + (two + 130 * U) * vi.abs(), A.abs())
        da[i] = s * mm(vi.t(), xi)
        dae[i] = s * mm((vei + (n + 66) * U * vi.abs()).t(), xi.abs())
        db[i] = s * mm(dyi.t(), ui)
        dbe[i] = s * mm(dyi.abs().t(), uei + (n + 66) * U * ui.abs())
    half = HALF.get(d["x"].dtype, 0.0)
    return dict(u=(u, ue), y=(y, ye + half * y.abs()), dx=(dx, dxe + half * dx.abs()), da=(da, dae), db=(db, dbe))


def check(got, want, label):
    w, tol = want
    err = (got.double() - w).abs()
    assert torch.isfinite(got).all(), label
    bad = err > tol + 1e-30
    assert not bad.any(), (label, int(bad.sum()), (err / (tol + 1e-30)).max().item())


def run(d, plan=None):
    plan = plan or fa.lora_pool_plan(d["index"], d["a"].shape[0])
    y, dx = d["y"].clone(), d["dx"].clone()
    u = fa.lora_pool_fwd(d["x"], d["a"], d["b"], y, d["scales"], plan)
    da, db = fa.lora_pool_bwd(d["x"], d["a"], d["b"], u, d["dy"], d["scales"], plan, dx=dx)
    return dict(u=u, y=y, da=da, db=db, dx=dx)


def run_and_check(d):
    got, want = run(d), exact(d)
    for k in got:
        check(got[k], want[k], k)
    none = (d["index"] < 0) | (d["index"] >= d["a"].shape[0])
    assert torch.equal(got["y"][none], d["y"][none]) and torch.equal(got["dx"][none], d["dx"][none])
    assert not got["u"][none].any()
    return got


SIZES = [  # T, L, K, M, r
    (1, 1, 1, 1, 1), (1, 3, 64, 96, 4), (2, 1, 8, 8, 16), (5, 9, 72, 40, 7), (16, 2, 128, 256, 16), (17, 4, 65, 130, 17),
    (63, 1, 515, 300, 8), (64, 1, 512, 512, 32), (65, 2, 100, 1001, 33), (200, 64, 256, 128, 16), (256, 1, 64, 64, 64),
    (257, 1, 130, 70, 12), (700, 3, 1001, 515, 48), (1500, 2, 768, 1536, 64), (33, 2048, 40, 24, 2),
    (2000, 700, 64, 72, 5),
]


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_64_bits(device, size, dt):
    run_and_check(make(*size, dt, seed=sum(size)))


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("index", ["none", "one", "ends", "runs", "outside"])
def test_indices(device, index, dt):
    """No token with an adapter; all with one; a first and last token alone; whole
    requests; indices far outside the pool."""
    T, L = 530, 6
    t = torch.arange(T, device="cuda")
    idx = dict(none=torch.full_like(t, -1), one=torch.full_like(t, 3), ends=torch.where((t == 0) | (t == T - 1), 2, 9),
               runs=t // 100, outside=torch.where(t % 3 == 0, 2 ** 31 - 1, torch.where(t % 3 == 1, -2 ** 31, t % L)))
    got = run_and_check(make(T, L, 200, 136, 16, dt, index=idx[index].to(torch.int32), seed=4))
    if index == "none":
        assert not got["da"].any() and not got["db"].any()


@pytest.mark.parametrize("T,L,order", [(70000, 5, "mixed"), (20000, 2048, "mixed"), (40000, 40, "runs")])
def test_plan_of_many_tokens(device, T, L, order):
    """The sums of a long batch by integers: every product and sum is exact in
    f32, so every result has to be equal to the exact one."""
    g = torch.Generator(device="cuda").manual_seed(1)
    if order == "mixed":
        idx = torch.randint(-1, L + 1, (T,), generator=g, device="cuda")
    else:
        idx = torch.randint(0, L, (T // 50,), generator=g, device="cuda").repeat_interleave(50)
    d = make(T, L, 8, 8, 2, BF, index=idx.to(torch.int32))
    for k in ("x", "a", "b", "y", "dy", "dx"):
        d[k] = torch.randint(-1, 2, d[k].shape, generator=g, device="cuda").to(BF)
    d["scales"].fill_(1.0)
    got, want = run(d), exact(d)
    for k in got:
        assert torch.equal(got[k].double(), want[k][0]), k


def test_same_bits_again_and_by_plan_memory(device):
    d = make(900, 7, 520, 264, 16, BF, seed=11)
    first = run(d)
    plan = fa.lora_pool_plan(torch.full_like(d["index"], 2), 7).update(d["index"])
    for again in (run(d), run(d, plan)):
        assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dt", [BF, F32])
def test_one_adapter_alone_has_the_same_result(device, dt):
    """A token's result does not depend on the pool beside it."""
    d = make(300, 4, 384, 200, 8, dt, seed=13)
    want = exact(d)
    e = dict(d, a=d["a"][2:3].contiguous(), b=d["b"][2:3].contiguous(), scales=d["scales"][2:3].contiguous(),
             index=torch.where(d["index"] == 2, 0, -1).to(torch.int32))
    got = run_and_check(e)
    rows = d["index"] == 2
    check(got["y"][rows], tuple(t[rows] for t in want["y"]), "y")
    check(got["da"][0], tuple(t[2] for t in want["da"]), "da")


@pytest.mark.parametrize("dt", [BF, F32])
def test_row_strides(device, dt):
    """Column slices at odd offsets; what lies beside them stays."""
    T, K, M = 130, 203, 77
    d = make(T, 3, K, M, 6, dt, seed=17)
    want = run_and_check(d)
    wide = lambda t, off: torch.full((T, t.shape[1] + 21), 7.0, dtype=dt, device="cuda")[:, off:off + t.shape[1]].copy_(t)
    plan = fa.lora_pool_plan(d["index"], 3)
    x, y, dy, dx = wide(d["x"], 3), wide(d["y"], 5), wide(d["dy"], 1), wide(d["dx"], 9)
    u = fa.lora_pool_fwd(x, d["a"], d["b"], y, d["scales"], plan)
    da, db = fa.lora_pool_bwd(x, d["a"], d["b"], u, dy, d["scales"], plan, dx=dx)
    for k, t in (("u", u), ("y", y), ("da", da), ("db", db), ("dx", dx)):
        assert torch.equal(t, want[k]), k
    for t, off, n in ((y, 5, M), (dx, 9, K)):
        assert (t._base[:, :off] == 7).all() and (t._base[:, off + n:] == 7).all()


@pytest.mark.parametrize("dt", [BF, F32])
def test_poison_stays_with_its_token_and_adapter(device, dt):
    """NaN in one token's rows and in one adapter's factors reaches only what is
    computed from them."""
    d = make(150, 5, 96, 80, 8, dt, seed=19)
    clean = run(d)
    bad = (d["index"] == 1).nonzero().flatten()[0]
    x, dy, a, b = (d[k].clone() for k in ("x", "dy", "a", "b"))
    x[bad], dy[bad] = float("nan"), float("inf")
    a[3], b[3] = float("nan"), float("nan")
    none = (d["index"] < 0).nonzero().flatten()
    x[none], dy[none] = float("nan"), float("nan")
    got = run(dict(d, x=x, dy=dy, a=a, b=b))
    fine = (d["index"] != 3) & (torch.arange(150, device="cuda") != bad)
    for k in ("y", "u", "dx"):
        assert torch.equal(got[k][fine], clean[k][fine]), k
    for k in ("da", "db"):
        assert torch.equal(got[k][[0, 2, 4]], clean[k][[0, 2, 4]]), k
    assert got["y"][bad].isnan().all()


def test_padded_ranks(device):
    """An adapter of rank 5 in a pool of rank 16: zeros in, zero gradients out."""
    d = make(200, 3, 160, 144, 16, BF, seed=23)
    d["a"][1, 5:], d["b"][1, :, 5:] = 0, 0
    got = run_and_check(d)
    assert not got["da"][1, 5:].any() and not got["db"][1, :, 5:].any()


def test_no_tokens_and_frozen_factors(device):
    d = make(0, 3, 64, 32, 4, BF)
    got = run(d)
    assert got["u"].shape == (0, 4) and not got["da"].any() and not got["db"].any()
    d = make(90, 3, 64, 32, 4, BF, seed=2)
    want = run(d)
    plan = fa.lora_pool_plan(d["index"], 3)
    dx = d["dx"].clone()
    assert fa.lora_pool_bwd(d["x"], d["a"], d["b"], want["u"], d["dy"], d["scales"], plan, dx=dx,
                            want_factors=False) == (None, None)
    assert torch.equal(dx, want["dx"])
    da, db = fa.lora_pool_bwd(d["x"], d["a"], d["b"], want["u"], d["dy"], d["scales"], plan)
    assert torch.equal(da, want["da"]) and torch.equal(db, want["db"])


@pytest.mark.parametrize("dt", [BF, F32])
def test_parts_of_the_backward(device, dt):
    """The gradients alone and dx alone have the whole backward's bits, where v
    comes in parts (wide dy) and where dx is narrower or wider than the factors."""
    for K, M in ((40, 1030), (1030, 300), (2100, 2100)):
        d = make(300, 3, K, M, 20, dt, seed=K)
        want = run_and_check(d)
        plan = fa.lora_pool_plan(d["index"], 3)
        da, db = fa.lora_pool_bwd(d["x"], d["a"], d["b"], want["u"], d["dy"], d["scales"], plan)
        assert torch.equal(da, want["da"]) and torch.equal(db, want["db"])
        dx = d["dx"].clone()
        fa.lora_pool_bwd(d["x"], d["a"], d["b"], want["u"], d["dy"], d["scales"], plan, dx=dx, want_factors=False)
        assert torch.equal(dx, want["dx"])


def test_autograd_matches_differences(device):
    """The wrapper's gradients against central differences in 64 bits (h = 1e-4)."""
    d = make(12, 3, 20, 10, 4, F32, seed=29)
    leaves = {k: d[k].clone().requires_grad_() for k in ("x", "a", "b", "y")}
    plan = fa.lora_pool_plan(d["index"], 3)
    out = fa.lora_pool(leaves["x"].view(3, 4, 20), leaves["a"], leaves["b"], leaves["y"].view(3, 4, 10), d["scales"],
                       plan)
    out.backward(d["dy"].view(3, 4, 10))

    def loss(vals):
        e = exact(dict(d, **vals))
        return (e["y"][0] * d["dy"].double()).sum().item()

    h = 1e-4
    for k, at in (("x", (0, 3)), ("x", (7, 19)), ("a", (1, 2, 5)), ("a", (2, 3, 0)), ("b", (0, 9, 1)), ("y", (11, 4))):
        lo, hi = d[k].double(), d[k].double()
        lo[at] -= h
        hi[at] += h
        want = (loss({k: hi}) - loss({k: lo})) / (2 * h)
        assert abs(leaves[k].grad[at].item() - want) < 1e-4 * (1 + abs(want)), (k, at)


@pytest.mark.parametrize("layout", ["expanded", "transposed"])
def test_autograd_of_inputs_without_rows(device, layout):
    """A broadcast or transposed x, base and upstream gradient: what a copy gives."""
    d = make(30, 3, 24, 24, 4, F32, seed=31)
    view = (lambda t: t[:1].expand(30, 24)) if layout == "expanded" else (lambda t: t[:24].t().contiguous().t())
    index = d["index"] if layout == "expanded" else d["index"][:24].contiguous()
    plan, got = fa.lora_pool_plan(index, 3), []
    for lay in (view, lambda t: view(t).contiguous()):
        x, a, b, y = (d[k].clone().requires_grad_() for k in ("x", "a", "b", "y"))
        out = fa.lora_pool(lay(x), a, b, lay(y), d["scales"], plan)
        out.backward(lay(d["dy"]))
        got.append([out, x.grad, a.grad, b.grad, y.grad])
    assert all(torch.equal(p, q) for p, q in zip(got[0][:4], got[1])) and got[0][1].any()
    # base's gradient is the upstream one itself, which autograd sums over a broadcast's 30 rows in an order that
    # follows the layout: n additions err by (n - 1) 2^-24 of the sum of magnitudes at most, in either order
    p, q = got[0][4], got[1][4]
    mags = torch.zeros_like(p).copy_(view(d["dy"]).abs().sum(0) if layout == "expanded" else view(d["dy"]).abs().sum())
    assert ((p - q).abs() <= 2 * 29 * 2.0 ** -24 * mags * (1 + 1e-5)).all()


def test_plan_changed_before_the_backward(device):
    d = make(12, 3, 20, 10, 4, F32, seed=29)
    plan = fa.lora_pool_plan(d["index"], 3)
    out = fa.lora_pool(d["x"].requires_grad_(), d["a"], d["b"], d["y"], d["scales"], plan)
    plan.update(torch.zeros_like(d["index"]))
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


def test_stream_and_graph(device):
    """On another stream, and captured: a replay sorts the index as it then is."""
    d = make(333, 6, 264, 520, 16, BF, seed=31)
    want = run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(d)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], want[k]) for k in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(d)
    for k in range(4):
        d["index"].copy_(torch.roll(d["index"], 37))
        d["x"].mul_(-1.125)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(d)
        assert all(torch.equal(outs[n], eager[n]) for n in eager), k


@pytest.mark.parametrize("dt", [BF, F32])
def test_infinities_come_through(device, dt):
    """An infinite activation of one token, rank 1: infinite where the formula
    says so, NaN nowhere else, and the other tokens as they were."""
    d = make(40, 2, 30, 24, 1, dt, seed=37)
    t = (d["index"] == 1).nonzero().flatten()[0]
    d["a"][1].abs_().add_(0.125)
    d["b"][1].abs_().add_(0.125)
    clean = run(d)
    d["x"] = d["x"].clone()
    d["x"][t] = d["x"][t].abs()
    d["x"][t, 7] = float("inf")
    got = run(d)
    assert (got["u"][t] == float("inf")).all() and (got["y"][t] == float("inf")).all()
    rest = torch.arange(40, device="cuda") != t
    for k in ("u", "y", "dx"):
        assert torch.equal(got[k][rest], clean[k][rest]), k
    assert torch.equal(got["da"][0], clean["da"][0]) and torch.equal(got["db"][0], clean["db"][0])


def test_wrappers_without_tokens(device):
    d = make(0, 2, 16, 8, 4, F32)
    leaves = {k: d[k].requires_grad_() for k in ("x", "a", "b")}
    out = fa.lora_pool(leaves["x"].view(0, 1, 16), leaves["a"], leaves["b"], d["y"].view(0, 1, 8), d["scales"],
                       fa.lora_pool_plan(d["index"], 2))
    out.sum().backward()
    assert leaves["x"].grad.shape == (0, 16) and not leaves["a"].grad.any() and not leaves["b"].grad.any()


def test_y_over_x(device):
    """y may be x itself where the widths agree: x is read first."""
    d = make(100, 3, 48, 48, 8, BF, seed=41)
    want = dict(d, y=d["x"].clone())
    plan = fa.lora_pool_plan(d["index"], 3)
    u0 = fa.lora_pool_fwd(d["x"], d["a"], d["b"], want["y"], d["scales"], plan)
    x = d["x"].clone()
    u1 = fa.lora_pool_fwd(x, d["a"], d["b"], x, d["scales"], plan)
    assert torch.equal(x, want["y"]) and torch.equal(u0, u1)


def test_memory_that_is_no_plan(device):
    """Whatever lies in the plan's memory, nothing outside the call's tensors is
    touched (the checks on every word of it are the host's arithmetic: indices
    are compared as unsigned against the sizes before any use)."""
    d = make(70, 3, 40, 24, 4, F32, seed=43)
    plan = fa.lora_pool_plan(d["index"], 3)
    words = plan.data.view(torch.int32)
    other = fa.lora_pool_plan(torch.zeros(69, dtype=torch.int32, device="cuda"), 3)
    words.zero_()  # sizes that are not the call's: nothing is done
    y = d["y"].clone()
    fa.lora_pool_fwd(d["x"], d["a"], d["b"], y, d["scales"], plan)
    assert torch.equal(y, d["y"])
    with pytest.raises(fa.FoundryAttnError):
        fa.lora_pool_fwd(d["x"], d["a"], d["b"], y, d["scales"], other)
