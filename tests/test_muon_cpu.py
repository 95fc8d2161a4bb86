"""What the orthogonalised step refuses, before any device work."""
import ctypes

import pytest
import torch

from foundry_attn import FoundryAttnError, _abi
from foundry_attn import block as fb
from foundry_attn._abi import lib

FAKE = 1 << 20


def args(**kw):
    a = _abi.MuonArgs(dtype=0, count=2, rows=16, cols=300, param=FAKE, grad=FAKE, momentum=FAKE, lr=0.02, beta=0.95,
                      weight_decay=0.1, eps=1e-7, scale=1.0, a=3.4445, b=-4.775, c=2.0315, steps=5, nesterov=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def call(*items, ws=FAKE, size=1 << 30):
    arr = (_abi.MuonArgs * len(items))(*items)
    return lib().fa_muon_step_many(arr, len(items), ws, size, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on fake pointers")
def test_calls_in_order_reach_the_device_check():
    assert call(args()) == call(args(), args(rows=300, cols=16, scale=4.0)) == _abi.FA_ERR_NO_DEVICE
    assert call(args(steps=0, lr=0.0, beta=0.0, nesterov=0)) == _abi.FA_ERR_NO_DEVICE


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 1), (dict(count=0), 1), (dict(rows=0), 1), (dict(cols=-4), 1), (dict(rows=65, cols=65), 2),
    (dict(cols=(1 << 30) + 1), 2), (dict(param=None), 1), (dict(param=FAKE + 1), 1), (dict(grad=None), 1),
    (dict(grad=FAKE + 2), 1), (dict(momentum=None), 1), (dict(lr=-1.0), 1), (dict(lr=float("inf")), 1),
    (dict(lr=float("nan")), 1), (dict(beta=1.0), 1), (dict(beta=-0.1), 1), (dict(weight_decay=-1.0), 1),
    (dict(lr=1.0, weight_decay=1.5), 1), (dict(eps=0.0), 1), (dict(eps=1e-301), 1), (dict(eps=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(a=float("nan")), 1), (dict(steps=-1), 1), (dict(steps=11), 1),
    (dict(count=1 << 30), 2),
])
def test_refusals(kw, code):
    assert call(args(**kw)) == code
    assert lib().fa_last_error()


@pytest.mark.parametrize("kw", [dict(dtype=1), dict(lr=0.1), dict(beta=0.9), dict(weight_decay=0.0), dict(eps=1e-6),
                                dict(a=1.0), dict(steps=4), dict(nesterov=0)])
def test_tensors_of_a_step_agree(kw):
    assert call(args(), args(**kw)) == _abi.FA_ERR_INVALID_ARG


def test_workspace():
    size = lambda *items: lib().fa_muon_step_many_workspace_size((_abi.MuonArgs * len(items))(*items), len(items))
    one = size(args())
    assert one > 0 and size(args(), args()) > one
    assert size(args(rows=0)) == size(args(rows=99, cols=99)) == 0
    assert lib().fa_muon_step_many_workspace_size(None, 1) == 0
    assert call(args(), size=one - 1) == call(args(), ws=None) == call(args(), ws=FAKE + 8) == _abi.FA_ERR_INVALID_ARG
    assert lib().fa_muon_step_many(None, 1, FAKE, 1 << 30, None) == _abi.FA_ERR_INVALID_ARG


def test_python_refusals():
    t = torch.zeros(4, 8)
    with pytest.raises(FoundryAttnError):
        fb.muon_step(t, t, t)
    with pytest.raises(FoundryAttnError):
        fb.muon_step(t.half(), t, t)
