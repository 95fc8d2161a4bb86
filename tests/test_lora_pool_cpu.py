"""What the pool of adapters refuses, before any device work."""
import ctypes

import pytest
import torch

import foundry_attn as fa
from foundry_attn import FoundryAttnError, _abi
from foundry_attn._abi import lib

FAKE = 1 << 20


def args(**kw):
    a = _abi.LoraPoolArgs(dtype=0, tokens=40, in_features=33, out_features=17, rank=5, adapters=3, x=FAKE, ldx=33,
                          a=FAKE, b=FAKE, scale=FAKE, plan=FAKE, plan_bytes=1 << 20, u=FAKE, y=FAKE, ldy=20,
                          workspace=FAKE, workspace_bytes=1 << 28)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def bwd_args(fwd=None, **kw):
    a = _abi.LoraPoolBwdArgs(fwd=args(**(fwd or {})), dy=FAKE, ldy=17, da=FAKE, db=FAKE, dx=2 * FAKE, ldx=33)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


fwd = lambda **kw: lib().fa_lora_pool_fwd(ctypes.byref(args(**kw)), None)
bwd = lambda f=None, **kw: lib().fa_lora_pool_bwd(ctypes.byref(bwd_args(f, **kw)), None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on fake pointers")
def test_calls_in_order_reach_the_device_check():
    assert fwd() == fwd(tokens=1, ldx=0) == fwd(rank=64, adapters=2048) == _abi.FA_ERR_NO_DEVICE
    assert fwd(tokens=0, x=None, y=None, u=None) == bwd(dict(tokens=0, x=None, u=None), dy=None) == _abi.FA_ERR_NO_DEVICE
    assert bwd() == bwd(dx=None) == bwd(da=None, db=None) == bwd(da=None, db=None, dx=FAKE) == _abi.FA_ERR_NO_DEVICE
    assert lib().fa_lora_pool_plan(FAKE, 40, 3, FAKE, 1 << 20, None) == _abi.FA_ERR_NO_DEVICE
    assert lib().fa_lora_pool_plan(None, 0, 3, FAKE, 1 << 20, None) == _abi.FA_ERR_NO_DEVICE


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(tokens=-1), dict(tokens=(1 << 28) + 1), dict(in_features=0), dict(in_features=(1 << 22) + 1),
    dict(out_features=0), dict(rank=0), dict(rank=65), dict(adapters=0), dict(adapters=2049), dict(x=None),
    dict(x=FAKE + 1), dict(ldx=32), dict(a=None), dict(b=FAKE + 1), dict(scale=None), dict(scale=FAKE + 2),
    dict(plan=None), dict(plan=FAKE + 8), dict(plan_bytes=100), dict(u=None), dict(u=FAKE + 2),
], ids=str)
def test_refusals_of_both(kw):
    assert fwd(**kw) == bwd(kw) == _abi.FA_ERR_INVALID_ARG
    assert lib().fa_last_error()


def test_refusals_of_one():
    bad = _abi.FA_ERR_INVALID_ARG
    assert fwd(y=None) == fwd(ldy=16) == bad
    assert fwd(in_features=1 << 20, ldx=1 << 20, workspace=None) == fwd(in_features=1 << 20, ldx=1 << 20,
                                                                        workspace_bytes=16) == bad
    assert bwd(dy=None) == bwd(ldy=16) == bwd(da=None) == bwd(db=FAKE + 1) == bwd(ldx=32) == bad
    assert bwd(dx=FAKE) == bwd(dict(x=2 * FAKE)) == bad  # dx over dy, over x
    assert bwd(dict(workspace=None)) == bwd(dict(workspace=FAKE + 64)) == bwd(dict(workspace_bytes=64)) == bad
    assert lib().fa_lora_pool_fwd(None, None) == lib().fa_lora_pool_bwd(None, None) == bad


@pytest.mark.parametrize("a", [(FAKE, -1, 3, FAKE, 1 << 20), (FAKE, 4, 0, FAKE, 1 << 20), (FAKE, 4, 2049, FAKE, 1 << 30),
                               (None, 4, 3, FAKE, 1 << 20), (FAKE + 1, 4, 3, FAKE, 1 << 20), (FAKE, 4, 3, None, 1 << 20),
                               (FAKE, 4, 3, FAKE + 8, 1 << 20), (FAKE, 400, 3, FAKE, 500)])
def test_plan_refusals(a):
    assert lib().fa_lora_pool_plan(*a, None) == _abi.FA_ERR_INVALID_ARG


def test_sizes():
    size = lib().fa_lora_pool_plan_size
    assert size(-1, 3) == size(4, 0) == size(4, 2049) == 0 < size(0, 1) <= size(1, 1) < size(1 << 28, 2048)
    for t in (0, 1, 1 << 28):
        a = args(tokens=t)
        assert lib().fa_lora_pool_fwd_workspace_size(ctypes.byref(a)) >= 0
        assert lib().fa_lora_pool_bwd_workspace_size(ctypes.byref(bwd_args(dict(tokens=t)))) >= t * 5 * 4
    assert lib().fa_lora_pool_fwd_workspace_size(None) == lib().fa_lora_pool_bwd_workspace_size(None) == 0


def test_python_refusals():
    i, x, a, b, y, s = (torch.zeros(4, dtype=torch.int32), torch.zeros(4, 8), torch.zeros(2, 3, 8),
                        torch.zeros(2, 6, 3), torch.zeros(4, 6), torch.ones(2))
    with pytest.raises(FoundryAttnError):
        fa.lora_pool_plan(i, 2)
    with pytest.raises(FoundryAttnError):
        fa.lora_pool_fwd(x, a, b, y, s, fa.LoraPoolPlan(4, 2, i))
