"""The C entry points of the gated norm answer bad arguments by a status, before any GPU call; the torch module refuses tensors that are
not on the GPU."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE = 1, 3
P = 4096   # an address that is never read: every call here ends in its checks


def desc(**changes):
    from geo_amd import _native
    d = _native.GatedNormDesc(struct_bytes=ctypes.sizeof(_native.GatedNormDesc), x=P, residual=P, weight=P, post_weight=P, gate=P,
                              residual_scale=P, rows=6, cols=8, x_stride=8, residual_stride=8, rows_per_gate=3, eps=1e-6, dtype=1)
    for k, v in changes.items():
        setattr(d, k, v)
    return ctypes.byref(d)


@pytest.fixture(scope="module")
def lib():
    from geo_amd import _native
    return _native.lib()


BAD = [dict(struct_bytes=8), dict(x=None), dict(residual=None), dict(weight=None), dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(cols=1 << 31),
       dict(x_stride=-1), dict(residual_stride=-1), dict(rows_per_gate=0), dict(rows_per_gate=4), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=3)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_descriptions(lib, bad):
    assert lib.geo_sc_gated_norm(desc(**bad), P, P, None, None) == INVALID
    assert lib.geo_sc_gated_norm_q8(desc(**bad), P, 8, P, P, None, 0, None) == INVALID
    assert lib.geo_sc_gated_norm_backward(desc(**bad), P, 8, P, 8, P, P, P, P, P, P, P, P, 1 << 30, None) == INVALID


def test_forward_refuses(lib):
    assert lib.geo_sc_gated_norm(None, P, P, None, None) == INVALID
    assert lib.geo_sc_gated_norm(desc(), None, P, None, None) == INVALID
    assert lib.geo_sc_gated_norm(desc(), P, None, None, None) == INVALID
    good = [P, 8, P, P, None, 0, None]
    for at, bad in ((0, None), (1, 7), (2, None), (3, None)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_gated_norm_q8(desc(), *args) == INVALID, (at, bad)
    assert lib.geo_sc_gated_norm_q8(desc(), P, 8, P, P, P, 5, None) == INVALID
    # no rows: nothing to do
    assert lib.geo_sc_gated_norm(desc(rows=0, x=None), None, None, None, None) == 0
    assert lib.geo_sc_gated_norm_q8(desc(rows=0, x=None), None, 8, None, None, None, 0, None) == 0


def test_backward_refuses(lib):
    size = ctypes.c_size_t()
    assert lib.geo_sc_gated_norm_backward_workspace_size(6, 8, ctypes.byref(size)) == 0 and size.value >= 5 * 8 * 4
    for rows, cols in ((0, 8), (6, 0), (1 << 31, 8)):
        assert lib.geo_sc_gated_norm_backward_workspace_size(rows, cols, ctypes.byref(size)) == INVALID
    assert lib.geo_sc_gated_norm_backward_workspace_size(6, 8, None) == INVALID
    good = [P, 8, P, 8, P, P, P, P, P, P, P, P, 1 << 30, None]
    for at, bad, status in ((0, None, INVALID), (1, -1, INVALID), (3, -1, INVALID), (4, None, INVALID), (5, None, INVALID), (6, None, INVALID),
                            (11, None, WORKSPACE), (11, P + 2, WORKSPACE), (12, 8, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_gated_norm_backward(desc(), *args) == status, (at, bad)
    for missing in ("post_weight", "gate", "residual_scale"):   # the gradient of what is not there
        assert lib.geo_sc_gated_norm_backward(desc(**{missing: None}), *good) == INVALID
    assert lib.geo_sc_gated_norm_backward(desc(rows=0), *good) == INVALID


def test_host_tensors_are_refused():
    from geo_amd import utils_functional as uf
    x = torch.zeros(2, 4)
    for call in (lambda: uf.gated_norm(x, x, x[0]), lambda: uf.gated_norm_q8(x, x, x[0])):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            call()
