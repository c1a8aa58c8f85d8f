"""The description of a gated norm from a caller built before it had `rstd`: taken as it is, and that field not read."""
import ctypes

import pytest
import torch

INVALID = 1
P = 4096   # an address that is never read


def desc(**changes):
    from geo_amd import _native
    d = _native.GatedNormDesc(struct_bytes=ctypes.sizeof(_native.GatedNormDesc), x=P, residual=P, weight=P, rows=0, cols=8, x_stride=8,
                              residual_stride=8, rows_per_gate=1, eps=1e-6, dtype=0)
    for k, v in changes.items():
        setattr(d, k, v)
    return d


def test_sizes():
    from geo_amd import _native
    lib, before = _native.lib(), _native.GatedNormDesc.rstd.offset
    for size, status in ((before, 0), (ctypes.sizeof(_native.GatedNormDesc), 0), (before - 8, INVALID), (before + 4, INVALID), (before + 16, INVALID)):
        d = ctypes.byref(desc(struct_bytes=size))
        assert lib.geo_sc_gated_norm(d, None, None, None, None) == status, size
        assert lib.geo_sc_gated_norm_q8(d, None, 8, None, None, None, 0, None) == status, size


@pytest.mark.gpu
def test_field():
    from geo_amd import _native
    lib, before = _native.lib(), _native.GatedNormDesc.rstd.offset
    x, w = torch.randn(6, 8, device="cuda"), torch.ones(8, device="cuda")
    want = ((x + x).square().mean(1) + 1e-6).rsqrt()
    for size in (before, ctypes.sizeof(_native.GatedNormDesc)):
        q, scale = torch.zeros(6, 16, dtype=torch.int8, device="cuda"), torch.zeros(6, device="cuda")
        total, rstd = torch.zeros(6, 8, device="cuda"), torch.full((6, 2), 7.0, device="cuda")
        d = desc(struct_bytes=size, x=x.data_ptr(), residual=x.data_ptr(), weight=w.data_ptr(), rows=6, rstd=rstd.data_ptr())
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.geo_sc_gated_norm_q8(ctypes.byref(d), q.data_ptr(), 16, scale.data_ptr(), total.data_ptr(), None, 0, stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(total, x + x) and (scale > 0).all()
        if size == before:
            assert (rstd == 7).all()
        else:   # no norm behind the block: 1; eight squares, their mean and a root: some 16 units
            assert (rstd[:, 0] == 1).all() and ((rstd[:, 1] / want - 1).abs() <= 16 * 2.0 ** -24).all()
