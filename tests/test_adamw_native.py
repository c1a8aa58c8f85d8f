"""The C entry point of the AdamW step answers bad arguments by a status, before any GPU call; the torch module refuses tensors that are
not on the GPU; the optimiser refuses its arguments."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE, UNSUPPORTED = 1, 3, 5
P = 4096   # an address that is never read: every call here ends in its checks


def call(tensor=None, options=None, count=1, workspace=None, workspace_bytes=0, struct_bytes=None):
    from geo_amd import _native
    t = _native.AdamWTensor(param=P, grad=P, exp_avg=P, exp_avg_sq=P, avg_scale=P, sq_scale=P, elements=10)
    o = _native.AdamWOptions(struct_bytes=ctypes.sizeof(_native.AdamWOptions) if struct_bytes is None else struct_bytes, state_bits=32, lr=1e-3,
                             beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, lo=-1, hi=1, step=1)
    for k, v in (tensor or {}).items():
        setattr(t, k, v)
    for k, v in (options or {}).items():
        setattr(o, k, v)
    return _native.lib().geo_sc_adamw(count, ctypes.byref(t), ctypes.byref(o), workspace, workspace_bytes, None)


NAN = float("nan")


@pytest.mark.parametrize("tensor", [dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(elements=-1),
                                    dict(copy=P)], ids=str)
def test_tensors(tensor):
    assert call(tensor, dict(copy_dtype=3)) == INVALID


@pytest.mark.parametrize("options", [dict(param_dtype=3), dict(grad_dtype=-1), dict(state_bits=16), dict(lr=-1.0), dict(lr=NAN), dict(beta1=1.0),
                                     dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=NAN), dict(eps=-1e-9), dict(weight_decay=-1.0), dict(lo=2.0),
                                     dict(step=0)], ids=str)
def test_options(options):
    assert call(None, options) == INVALID


def test_more_refusals():
    from geo_amd import _native
    assert call(count=-1) == INVALID and call(struct_bytes=8) == INVALID
    for scale in ("avg_scale", "sq_scale"):
        assert call({scale: None}, dict(state_bits=8)) == INVALID
    assert call(dict(elements=1 << 50)) == UNSUPPORTED
    for workspace, size in ((None, 16), (P, 8), (P + 4, 16)):
        assert call(None, dict(device_step=P, step=0), workspace=workspace, workspace_bytes=size) == WORKSPACE
    o = _native.AdamWOptions(struct_bytes=ctypes.sizeof(_native.AdamWOptions), state_bits=32, lr=1e-3, grad_scale=1.0, lo=-1, hi=1, step=1)
    assert _native.lib().geo_sc_adamw(1, None, ctypes.byref(o), None, 0, None) == INVALID
    assert _native.lib().geo_sc_adamw(0, None, None, None, 0, None) == INVALID


def test_nothing_to_do():
    assert call(count=0) == 0
    assert call(dict(elements=0, param=None, grad=None)) == 0


def test_host_tensors_are_refused():
    from geo_amd import utils_functional as uf
    t = [torch.zeros(4)]
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        uf.adamw_step(t, t, t, t, 1, 1e-3)
    with pytest.raises(RuntimeError, match="one length"):
        uf.adamw_step(t, [], t, t, 1, 1e-3)
    with pytest.raises(RuntimeError, match="1 or more"):
        uf.adamw_step(t, t, t, t, 0, 1e-3)
    uf.adamw_step([], [], [], [], 1, 1e-3)   # no tensors: nothing to do


def test_optimiser_refuses():
    from geo_amd import network
    p = [torch.zeros(4, requires_grad=True)]
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            network.AdamW(p, **bad)
        with pytest.raises(ValueError):
            network.AdamW([dict(params=p, **bad)])
