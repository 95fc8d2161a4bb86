"""The operators of many adapters over one frozen model, as timed cases.

Every case is one pass through the public entry points of foundry_attn
(own = True) or through the same formulas in elementary torch operations
(own = False):

  pool   the adapters of many requests beside one shared projection
         (ops.lora_pool_plan, lora_pool_fwd, lora_pool_bwd): token t belongs to
         adapter i = index[t], or to none where index[t] is outside the pool;
           u[t] = A_i x[t],  y[t] += s_i B_i u[t],
         and with train also
           v[t] = B_i^T dy[t],  dx[t] += s_i A_i^T v[t],
           dA_i = s_i sum_t v[t] x[t]^T,  dB_i = s_i sum_t dy[t] u[t]^T
  norm   layer norm with weight and bias (block.layer_norm_fwd) and, with
         train, its backward with the sums over the rows that are the weight's
         and the bias's gradients (block.layer_norm_bwd)
  muon   an optimiser step of low-rank factors (block.muon_step_many):
           m = beta m + g,  w = g + beta m,  X = w / (|w| + eps), `steps` times
           X = a X + (b X X^T + c (X X^T)^2) X,
           p = p (1 - lr wd) - lr sqrt(max(1, rows / cols)) X

listed() holds fixed cases, draw() further ones of the same ranges: from a
single decoded token to a batch of 8192, pools of one to 64 adapters of ranks
1 to 64, widths from 64 to 8192, odd ones among them, bf16 and f32.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
NORM_EPS = 1e-5
MUON = dict(lr=0.02, beta=0.95, weight_decay=0.01, eps=1e-7, a=3.4445, b=-4.7750, c=2.0315)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One request decodes one token: the call's latency.
        dict(name="pool_token", kind="pool", dtype="bf16", tokens=1, adapters=8, fin=2048, fout=2048, rank=16,
             order="mixed", train=False),
        # A decode step of 64 requests over 48 adapters, some without one.
        dict(name="pool_decode_64", kind="pool", dtype="bf16", tokens=64, adapters=48, fin=4096, fout=4096, rank=16,
             order="mixed", train=False),
        # Prompts of some tens of requests in one ragged batch, rank 32, into an MLP's width.
        dict(name="pool_prompts_6000", kind="pool", dtype="bf16", tokens=6000, adapters=12, fin=2048, fout=8192,
             rank=32, order="runs", train=False),
        # Sizes that nothing divides, f32, as a numerics check of the path runs it.
        dict(name="pool_odd_f32", kind="pool", dtype="f32", tokens=777, adapters=5, fin=1001, fout=515, rank=12,
             order="runs", train=True),
        # Four adapters trained side by side over one frozen projection.
        dict(name="pool_train_4096", kind="pool", dtype="bf16", tokens=4096, adapters=4, fin=4096, fout=4096, rank=16,
             order="runs", train=True),
        # A small batch whose samples lie in any order, rank 4.
        dict(name="pool_train_300", kind="pool", dtype="bf16", tokens=300, adapters=16, fin=768, fout=1536, rank=4,
             order="mixed", train=True),
        # The norm of a decode step.
        dict(name="norm_rows_8", kind="norm", dtype="bf16", rows=8, cols=2048, train=False),
        # A training batch at width 4096.
        dict(name="norm_train_4096", kind="norm", dtype="bf16", rows=4096, cols=4096, train=True),
        # Odd rows and columns in f32.
        dict(name="norm_odd_f32", kind="norm", dtype="f32", rows=1537, cols=1001, train=True),
        # Many short rows, a long batch.
        dict(name="norm_train_32768", kind="norm", dtype="bf16", rows=32768, cols=1024, train=True),
        # The two factors of one adapter.
        dict(name="muon_pair", kind="muon", dtype="bf16", count=1, rank=16, fin=4096, fout=4096, steps=5),
        # Every factor of a stack: 64 projections, rank 32, f32 factors.
        dict(name="muon_stack_64", kind="muon", dtype="f32", count=64, rank=32, fin=2048, fout=8192, steps=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 8 or more, now and then any."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 64 * 64 if rng.random() < 0.7 else n)


def draw(rng):
    kind = rng.choice(["pool", "pool", "pool", "norm", "norm", "muon", "muon"])
    if kind == "pool":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        case = dict(kind=kind, dtype=dtype, tokens=_log_int(rng, 1, 8192 if dtype == "bf16" else 1024),
                    adapters=_log_int(rng, 1, 64), fin=_width(rng, 64, 8192 if dtype == "bf16" else 2048),
                    fout=_width(rng, 64, 8192 if dtype == "bf16" else 2048),
                    rank=rng.choice([1, 4, 8, 8, 16, 16, 16, 24, 32, 64, 7]),
                    order=rng.choice(["runs", "mixed"]), train=rng.random() < 0.5)
        while _pool_cost(case) > 4.0e8:
            case["tokens"] = max(1, case["tokens"] // 2)
            case["adapters"] = max(1, case["adapters"] * 3 // 4)
        return case
    if kind == "norm":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        case = dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, 32768), cols=_width(rng, 64, 8192),
                    train=rng.random() < 0.7)
        while case["rows"] * case["cols"] > 32768 * 1024 // (1 if dtype == "bf16" else 2):
            case["rows"] = max(1, case["rows"] // 2)
        return case
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), count=_log_int(rng, 1, 64),
                rank=rng.choice([1, 4, 8, 16, 16, 32, 32, 64, 12]), fin=_width(rng, 64, 8192),
                fout=_width(rng, 64, 8192), steps=rng.choice([5, 5, 5, 3, 6]))
    while case["count"] * case["rank"] * (case["fin"] + case["fout"]) > 64 * 32 * 10240:
        case["count"] = max(1, case["count"] // 2)
    return case


def _pool_cost(case):
    """Bytes of the activations and, in training, of every adapter's gradients."""
    n = 2 if case["dtype"] == "bf16" else 4
    both = case["fin"] + case["fout"]
    acts = case["tokens"] * both * n * (3 if case["train"] else 1.5)
    return acts + case["adapters"] * case["rank"] * both * (4 if case["train"] else n)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _index(case, gen):
    """The adapter of each token: whole requests in a row ("runs") or token by
    token ("mixed"); about one request in ten has none (-1)."""
    t, n = case["tokens"], case["adapters"]
    if case["order"] == "mixed":
        idx = torch.randint(0, n, (t,), generator=gen, device=DEV)
        none = torch.rand(t, generator=gen, device=DEV) < 0.1
    else:
        cuts = min(t - 1, 3 * n)
        first = torch.zeros(t, dtype=torch.int64, device=DEV)
        if cuts > 0:
            first[torch.randint(1, t, (cuts,), generator=gen, device=DEV)] = 1
        run = first.cumsum(0)
        idx = torch.randint(0, n, (cuts + 1,), generator=gen, device=DEV)[run]
        none = (torch.rand(cuts + 1, generator=gen, device=DEV) < 0.1)[run]
    idx[none] = -1
    if t == 1:
        idx[0] = n // 2
    return idx.to(torch.int32)


def _prepare_pool(case, gen):
    dt = DTYPES[case["dtype"]]
    t, n, k, m, r = (case[f] for f in ("tokens", "adapters", "fin", "fout", "rank"))
    st = dict(index=_index(case, gen), x=_randn(gen, t, k, dtype=dt), y=_randn(gen, t, m, dtype=dt),
              a=_randn(gen, n, r, k, std=1 / math.sqrt(k), dtype=dt), b=_randn(gen, n, m, r, std=0.3 / math.sqrt(r),
                                                                                  dtype=dt),
              scales=0.5 + torch.rand(n, generator=gen, device=DEV))
    if case["train"]:
        st.update(dy=_randn(gen, t, m, dtype=dt), dx=_randn(gen, t, k, dtype=dt))
    return st


def _prepare_norm(case, gen):
    dt = DTYPES[case["dtype"]]
    n, c = case["rows"], case["cols"]
    scale = torch.exp(0.5 * torch.randn(n, 1, generator=gen, device=DEV))
    st = dict(x=((torch.randn(n, c, generator=gen, device=DEV) + 0.3) * scale).to(dt),
              weight=(1 + 0.1 * torch.randn(c, generator=gen, device=DEV)).to(dt),
              bias=_randn(gen, c, std=0.1, dtype=dt))
    if case["train"]:
        st["dy"] = _randn(gen, n, c, dtype=dt)
    return st


def _low_rank_noise(gen, *shape):
    """Gradients as they come: a few strong directions and noise around them."""
    u = torch.randn(*shape[:-1], 3, generator=gen, device=DEV)
    v = torch.randn(shape[0], 3, shape[-1], generator=gen, device=DEV)
    return 1e-3 * ((u[..., None] * v[:, None]).sum(-2) + 0.3 * torch.randn(*shape, generator=gen, device=DEV))


def _prepare_muon(case, gen):
    dt = DTYPES[case["dtype"]]
    n, r = case["count"], case["rank"]
    st = {}
    for f, shape in (("a", (n, r, case["fin"])), ("b", (n, case["fout"], r))):
        st["p" + f] = _randn(gen, *shape, std=0.05, dtype=dt)
        st["g" + f] = _low_rank_noise(gen, *shape)
        st["m" + f] = _low_rank_noise(gen, *shape)
    return st


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = {"pool": _prepare_pool, "norm": _prepare_norm, "muon": _prepare_muon}[case["kind"]](case, gen)
    st["case"] = case
    return st


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _calls():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "foundry-trainer_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import foundry_attn as fa
    from foundry_attn import block as fb
    return fa, fb


def _own_pool(st):
    fa, _ = _calls()
    case = st["case"]
    plan = fa.lora_pool_plan(st["index"], case["adapters"])
    u = fa.lora_pool_fwd(st["x"], st["a"], st["b"], st["y"], st["scales"], plan)
    if not case["train"]:
        return [st["y"], u]
    da, db = fa.lora_pool_bwd(st["x"], st["a"], st["b"], u, st["dy"], st["scales"], plan, dx=st["dx"])
    return [st["y"], u, da, db, st["dx"]]


def _own_norm(st):
    _, fb = _calls()
    y, mean, rstd = fb.layer_norm_fwd(st["x"], st["weight"], st["bias"], NORM_EPS)
    if not st["case"]["train"]:
        return [y, mean, rstd]
    return [y, mean, rstd, *fb.layer_norm_bwd(st["x"], st["dy"], st["weight"], mean, rstd)]


def _own_muon(st):
    _, fb = _calls()
    fb.muon_step_many([(st["p" + f], st["g" + f], st["m" + f]) for f in "ab"], lr=MUON["lr"], beta=MUON["beta"],
                      weight_decay=MUON["weight_decay"], steps=st["case"]["steps"], eps=MUON["eps"],
                      coeffs=(MUON["a"], MUON["b"], MUON["c"]))
    return [st["pa"], st["ma"], st["pb"], st["mb"]]


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_pool(st):
    """All adapters' products for all tokens, each token's own kept by a mask."""
    case = st["case"]
    t, n, k, m, r = (case[f] for f in ("tokens", "adapters", "fin", "fout", "rank"))
    x, a, b, sc = st["x"].float(), st["a"].float(), st["b"].float(), st["scales"]
    mine = (st["index"][:, None] == torch.arange(n, device=DEV)[None]).float()[:, :, None]  # [T, L, 1]
    rows_a = a.reshape(n * r, k)                      # [L r, K]
    cols_b = b.permute(0, 2, 1).reshape(n * r, m)     # [L r, M]
    us = (x @ rows_a.t()).reshape(t, n, r) * mine
    u = us.sum(1)
    scaled = (us * sc[None, :, None]).reshape(t, n * r)
    st["y"].copy_(st["y"].float() + scaled @ cols_b)
    if not case["train"]:
        return [st["y"], u]
    dy = st["dy"].float()
    vs = ((dy @ cols_b.t()).reshape(t, n, r) * mine * sc[None, :, None]).reshape(t, n * r)
    da = (vs.t() @ x).reshape(n, r, k)
    db = (scaled.t() @ dy).reshape(n, r, m).permute(0, 2, 1).contiguous()
    st["dx"].copy_(st["dx"].float() + vs @ rows_a)
    return [st["y"], u, da, db, st["dx"]]


def _plain_norm(st):
    x, w, b = st["x"].float(), st["weight"].float(), st["bias"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = torch.rsqrt((d * d).mean(1) + NORM_EPS)
    n = d * rstd[:, None]
    y = (n * w + b).to(st["x"].dtype)
    if not st["case"]["train"]:
        return [y, mean, rstd]
    dy = st["dy"].float()
    dn = dy * w
    dx = rstd[:, None] * (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True))
    return [y, mean, rstd, dx.to(st["x"].dtype), (dy * n).sum(0), dy.sum(0)]


def _plain_muon(st):
    out = []
    for f in "ab":
        p, g, m = st["p" + f], st["g" + f], st["m" + f]
        m.copy_(MUON["beta"] * m + g)
        w = g + MUON["beta"] * m
        x = w / ((w * w).sum((1, 2), keepdim=True).sqrt() + MUON["eps"])
        rows, cols = w.shape[1:]
        wide = rows <= cols
        x = x if wide else x.transpose(1, 2).contiguous()
        for _ in range(st["case"]["steps"]):
            s = x @ x.transpose(1, 2)
            x = MUON["a"] * x + (MUON["b"] * s + MUON["c"] * (s @ s)) @ x
        x = x if wide else x.transpose(1, 2)
        p.copy_(p.float() * (1 - MUON["lr"] * MUON["weight_decay"])
                - (MUON["lr"] * math.sqrt(max(1.0, rows / cols))) * x)
        out += [p, m]
    return out


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"pool": _own_pool, "norm": _own_norm, "muon": _own_muon}[kind](state)
    return {"pool": _plain_pool, "norm": _plain_norm, "muon": _plain_muon}[kind](state)


# ---------------------------------------------------------------------------
# the work of a pass, and its results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    n = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "pool":
        t, r, both = case["tokens"], case["rank"], case["fin"] + case["fout"]
        # factors that occur, each read once: about as many as there are tokens, at most all
        held = min(case["adapters"], t)
        size = t * (case["fin"] + 2 * case["fout"]) * n + held * r * both * n + t * (r + 1) * 4
        flops = 2.0 * t * r * both
        if case["train"]:
            size += t * (2 * case["fin"] + case["fout"]) * n + case["adapters"] * r * both * 4
            flops *= 3
        return {"bytes": float(size), "flops": flops}
    if case["kind"] == "norm":
        e, c = float(case["rows"]) * case["cols"], case["cols"]
        if case["train"]:
            return {"bytes": 4 * e * n + 2 * c * n + 8 * c + 8 * case["rows"], "flops": 20 * e}
        return {"bytes": 2 * e * n + 2 * c * n + 8 * case["rows"], "flops": 8 * e}
    e = float(case["count"]) * case["rank"] * (case["fin"] + case["fout"])
    r = case["rank"]
    return {"bytes": e * (2 * n + 12), "flops": e * (4.0 * r + 8) + 2 * case["count"] * 4.0 * case["steps"] * r ** 3}


def _exact_pool(case, st):
    n, r = case["adapters"], case["rank"]
    x, a, b, y = (st[f].double() for f in ("x", "a", "b", "y"))
    u = torch.zeros(case["tokens"], r, dtype=torch.float64, device=DEV)
    train = case["train"]
    if train:
        dy, dx = st["dy"].double(), st["dx"].double()
        da, db = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(n):
        rows = torch.nonzero(st["index"] == i).flatten()
        if not len(rows):
            continue
        s = float(st["scales"][i])
        u[rows] = torch.mm(x[rows], a[i].t().contiguous())
        y[rows] += s * torch.mm(u[rows], b[i].t().contiguous())
        if train:
            v = s * torch.mm(dy[rows], b[i])
            dx[rows] += torch.mm(v, a[i])
            da[i] = torch.mm(v.t().contiguous(), x[rows])
            db[i] = s * torch.mm(dy[rows].t().contiguous(), u[rows])
    return [y, u, da, db, dx] if train else [y, u]


def _exact_norm(case, st):
    x, w, b = (st[f].double() for f in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0)
    rstd = 1 / torch.sqrt(var + NORM_EPS)
    hat = (x - mean[:, None]) * rstd[:, None]
    y = torch.addcmul(b[None], hat, w[None])
    if not case["train"]:
        return [y, mean, rstd]
    dy = st["dy"].double()
    # the gradient through the normalisation: what is left of dy w outside the span of 1 and hat
    gw = dy * w
    c = case["cols"]
    along = (gw * hat).sum(1) / c
    dx = (gw - gw.sum(1)[:, None] / c - along[:, None] * hat) * rstd[:, None]
    return [y, mean, rstd, dx, (hat * dy).sum(0), dy.sum(0)]


def _exact_muon(case, st):
    """By the eigenvectors of w w^T: the products act on each singular value s
    of X alone, s -> s (a + b s^2 + c s^4)."""
    out = []
    for f in "ab":
        p, g, m = (st[k + f].double() for k in "pgm")
        m = MUON["beta"] * m + g
        w = g + MUON["beta"] * m
        rows, cols = w.shape[1:]
        short = w if rows <= cols else w.transpose(1, 2).contiguous()
        norm = w.flatten(1).norm(dim=1) + MUON["eps"]
        gram = torch.bmm(short, short.transpose(1, 2).contiguous()).cpu()
        val, vec = torch.linalg.eigh(gram)
        s2 = (val.clamp_min(0).to(DEV) / norm[:, None] ** 2)
        gain = torch.ones_like(s2)
        for _ in range(case["steps"]):
            q = MUON["a"] + MUON["b"] * s2 + MUON["c"] * s2 * s2
            gain, s2 = gain * q, s2 * q * q
        vec = vec.to(DEV)
        turn = torch.bmm(vec * (gain / norm[:, None])[:, None, :], vec.transpose(1, 2).contiguous())
        x = torch.bmm(turn, short)
        x = x if rows <= cols else x.transpose(1, 2)
        out += [p * (1 - MUON["lr"] * MUON["weight_decay"]) - MUON["lr"] * math.sqrt(max(1.0, rows / cols)) * x, m]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"pool": _exact_pool, "norm": _exact_norm, "muon": _exact_muon}[case["kind"]](case, st)
