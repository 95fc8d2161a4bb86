"""What the layer norm refuses, before any device work."""
import ctypes

import pytest
import torch

from foundry_attn import FoundryAttnError, _abi
from foundry_attn import block as fb
from foundry_attn._abi import lib

FAKE = 1 << 20


def fwd_args(**kw):
    a = _abi.LayerNormArgs(dtype=0, param_dtype=1, rows=5, cols=33, eps=1e-5, x=FAKE, ldx=33, weight=FAKE, bias=FAKE,
                           y=FAKE, ldy=40, mean=FAKE, rstd=FAKE)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def bwd_args(fwd=None, **kw):
    a = _abi.LayerNormBwdArgs(fwd=fwd_args(**(fwd or {})), dy=FAKE, lddy=33, dres=FAKE, ldres=33, dx=FAKE, lddx=33,
                              dweight=FAKE, dbias=FAKE, workspace=FAKE, workspace_bytes=1 << 24)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def ready():
    """What a call that is in order comes to here, without a GPU."""
    return _abi.FA_ERR_NO_DEVICE


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on fake pointers")
def test_calls_in_order_reach_the_device_check():
    assert lib().fa_layer_norm_fwd(ctypes.byref(fwd_args()), None) == ready()
    assert lib().fa_layer_norm_fwd(ctypes.byref(fwd_args(bias=None, mean=None, rstd=None)), None) == ready()
    assert lib().fa_layer_norm_fwd(ctypes.byref(fwd_args(rows=1, ldx=0)), None) == ready()
    assert lib().fa_layer_norm_bwd(ctypes.byref(bwd_args()), None) == ready()
    assert lib().fa_layer_norm_bwd(ctypes.byref(bwd_args(dweight=None, dbias=None, workspace=None)), None) == ready()


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), 1), (dict(param_dtype=-1), 1), (dict(rows=-1), 1), (dict(cols=0), 1), (dict(cols=32769), 2),
    (dict(x=None), 1), (dict(x=FAKE + 1), 1), (dict(ldx=32), 1), (dict(weight=None), 1), (dict(weight=FAKE + 2), 1),
])
def test_refusals_of_both(kw, code):
    assert lib().fa_layer_norm_fwd(ctypes.byref(fwd_args(**kw)), None) == code
    assert lib().fa_layer_norm_bwd(ctypes.byref(bwd_args(kw)), None) == code
    assert lib().fa_last_error()


@pytest.mark.parametrize("kw", [dict(eps=0.0), dict(eps=float("nan")), dict(y=None), dict(ldy=32), dict(bias=FAKE + 2),
                                dict(mean=None), dict(rstd=FAKE + 2)])
def test_forward_refusals(kw):
    assert lib().fa_layer_norm_fwd(ctypes.byref(fwd_args(**kw)), None) == _abi.FA_ERR_INVALID_ARG


@pytest.mark.parametrize("fwd,kw", [
    (dict(mean=None), {}), ({}, dict(dy=None)), ({}, dict(lddy=5)), ({}, dict(dx=None)), ({}, dict(ldres=1)),
    ({}, dict(dweight=FAKE + 1)), ({}, dict(workspace=None)), ({}, dict(workspace=FAKE + 8)),
    ({}, dict(workspace_bytes=8)),
])
def test_backward_refusals(fwd, kw):
    assert lib().fa_layer_norm_bwd(ctypes.byref(bwd_args(fwd, **kw)), None) == _abi.FA_ERR_INVALID_ARG


def test_null_and_sizes():
    assert lib().fa_layer_norm_fwd(None, None) == lib().fa_layer_norm_bwd(None, None) == _abi.FA_ERR_INVALID_ARG
    size = lambda **kw: lib().fa_layer_norm_bwd_workspace_size(ctypes.byref(bwd_args(kw)))
    assert lib().fa_layer_norm_bwd_workspace_size(None) == size(cols=0) == size(rows=-1) == size(rows=0) == 0
    assert size(rows=1 << 30, cols=32768) <= 1 << 30 and size() >= 33 * 8


def test_python_refuses_host_tensors():
    x, w = torch.ones(4, 8), torch.ones(8)
    with pytest.raises(FoundryAttnError):
        fb.layer_norm_fwd(x, w)
    with pytest.raises(FoundryAttnError):
        fb.layer_norm_bwd(x, x, w, w[:4], w[:4])
