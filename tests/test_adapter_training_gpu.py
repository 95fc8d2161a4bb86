"""The operators of adapter training together: a layer norm with a trained
weight and bias, a frozen projection of its output with a pool of adapters
beside it, the gradients through both, and the orthogonalised step of every
adapter's factors; and that step on the checkpointed stack of LoRA blocks.

Each step is checked by itself, from the parameters it began with: the gradients
against autograd of the formulas in 64 bits on the host (rel-L2 1e-4 in f32,
where the longest sum has 300 terms, 300 * 2^-24 of the absolute terms at most;
1e-2 in bf16, where the norm, the projection, the adapters and each gradient
round by 2^-8 of a value at most, 1.1e-3 root mean square, some six times in a
row), the step against its formulas from the gradients that it was given."""
import pytest
import torch

import foundry_attn as fa
from foundry_attn import block as fb
from foundry_attn import checkpoint as ck
from helpers import check_gate
from test_checkpoint_gpu import build, stack
from test_block_gpu import dev
from test_muon_gpu import exact as muon_exact

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
T, C, M, L, R = 300, 96, 160, 5, 8


def oracle(x, index, W, scales, dy, params):
    """Loss gradients in 64 bits on the host."""
    c = lambda t: t.detach().double().cpu()
    p = {k: c(v).requires_grad_() for k, v in params.items()}
    xx = c(x).requires_grad_()
    mean = xx.mean(1, keepdim=True)
    n = (xx - mean) / ((xx - mean).square().mean(1, keepdim=True) + 1e-5).sqrt() * p["w"] + p["b"]
    y = n @ c(W).t()
    idx = index.cpu().long()
    for i in range(L):
        rows = (idx == i)[:, None].double()
        y = y + rows * float(scales[i]) * (n @ p["A"][i].t() @ p["B"][i].t())
    (y * c(dy)).sum().backward()
    return y.detach(), {**{k: v.grad for k, v in p.items()}, "x": xx.grad}


@pytest.mark.parametrize("dt", [F32, BF])
def test_steps_of_many_adapters(device, dt):
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device="cuda")).to(dt)
    params = dict(w=(1 + 0.1 * rn(C).float()).to(dt), b=rn(C, std=0.1), A=rn(L, R, C, std=C ** -0.5),
                  B=rn(L, M, R, std=0.2))
    W, scales = rn(M, C, std=C ** -0.5), torch.linspace(0.5, 2.0, L, device="cuda")
    momenta = {k: torch.zeros(params[k].shape, device="cuda") for k in "AB"}
    for step in range(3):
        x, dy = rn(T, C), rn(T, M)
        index = torch.randint(-1, L, (T,), generator=g, device="cuda").to(torch.int32)
        index[index == step] = -1  # one adapter sits this step out
        leaves = {k: v.detach().requires_grad_() for k, v in params.items()}
        xx = x.detach().requires_grad_()
        plan = fa.lora_pool_plan(index, L)
        n = fb.layer_norm(xx, leaves["w"], leaves["b"])
        y = fa.lora_pool(n, leaves["A"], leaves["B"], torch.mm(n, W.t()), scales, plan)
        y.backward(dy)
        want_y, want = oracle(x, index, W, scales, dy, params)
        host = lambda t: t.detach().float().cpu().numpy()
        check_gate("y", host(y), want_y.numpy(), dt == BF)
        for k, leaf in {**leaves, "x": xx}.items():
            check_gate(f"d{k}", host(leaf.grad), want[k].numpy(), dt == BF)
        assert not leaves["A"].grad[step].any() and not leaves["B"].grad[step].any()
        grads = {k: leaves[k].grad.float() for k in "AB"}
        wants = {k: muon_exact(params[k], grads[k], momenta[k], 0.02, 0.95, 0.01, 5, True, 1e-7, fb.MUON_COEFFS, None)
                 for k in "AB"}
        with torch.no_grad():
            fb.muon_step_many([(params[k], grads[k], momenta[k]) for k in "AB"], lr=0.02, weight_decay=0.01)
        for k in "AB":
            wp, wm, tol = wants[k]
            half = 2.0 ** -8 if dt == BF else 2.0 ** -24
            err = (params[k].double().cpu() - wp).abs()
            assert (err <= tol + (half + 3 * 2.0 ** -24) * wp.abs() + half * tol).all(), (step, k)


@pytest.mark.parametrize("dt", [F32, BF])
def test_stack_step(device, dt):
    """checkpoint.apply_muon: every factor of the double and the single block
    takes its step, and what the blocks derive from the factors follows."""
    dcase, scase, targets = build(dt)
    st = stack(dcase, scase, dt)
    inputs = [dev(dcase["x"][n], dt) for n in ("txt", "img")]
    _, _, grads = ck.checkpointed_step(st, inputs, ck.mse_seed([dev(t, dt) for t in targets]))
    items = [it for k, s in enumerate(st) if grads.get(k) for it in s.block._factor_states(grads[k])]
    assert len(items) == 2 * (2 * 4 + 2)
    want = [muon_exact(p, g, m, 0.02, 0.95, 0.0, 5, True, 1e-7, fb.MUON_COEFFS, None) for p, g, m, _ in items]
    ck.apply_muon(st, grads)
    for (p, _, m, _), (wp, wm, tol) in zip(items, want):
        half = 2.0 ** -8 if dt == BF else 2.0 ** -24
        assert ((p.double().cpu() - wp).abs() <= tol + (half + 3 * 2.0 ** -24) * wp.abs() + half * tol).all()
    out = st[0].forward(inputs, False)[0][1].clone()
    st[0].block.refresh_adapters()
    assert torch.equal(out, st[0].forward(inputs, False)[0][1])
