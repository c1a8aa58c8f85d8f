"""The C entry points of the dense layers and of the distillation loss answer bad arguments by a status, before any GPU call; the
torch module refuses tensors that are not on the GPU; workspace queries."""
import ctypes

import pytest
import torch

INVALID, WORKSPACE = 1, 3


@pytest.fixture(scope="module")
def lib():
    from geo_amd import _native
    return _native.lib()


P = 4096   # an address that is never read: every call here ends in its checks


def test_quantize_rows_refuses(lib):
    good = [P, 0, 4, 8, 8, P, 8, P, None, 0, None]
    for at, bad in ((0, None), (1, 3), (2, -1), (2, 1 << 31), (3, 0), (3, 1 << 31), (4, -1), (5, None), (6, 7), (7, None)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_quantize_rows(*args) == INVALID, (at, bad)
    args = list(good)
    args[8], args[9] = P, 7          # values of no known type
    assert lib.geo_sc_quantize_rows(*args) == INVALID
    args = list(good)
    args[2] = 0
    assert lib.geo_sc_quantize_rows(*args) == 0   # no rows: nothing to do


def test_rms_norm_refuses(lib):
    good = [P, None, P, 1, 4, 8, 8, 8, 1e-6, P, 8, P, None, None, 0, None, None]
    for at, bad in ((0, None), (2, None), (3, -1), (4, -1), (5, 0), (6, -1), (7, -1), (8, -1.0), (8, float("nan")), (9, None), (10, 7), (11, None)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_rms_norm_q8(*args) == INVALID, (at, bad)
    size = ctypes.c_size_t()
    assert lib.geo_sc_rms_norm_q8_backward_workspace_size(100, 64, ctypes.byref(size)) == 0 and size.value >= 64 * 4
    assert lib.geo_sc_rms_norm_q8_backward_workspace_size(100, 0, ctypes.byref(size)) == INVALID
    good = [P, 1, 8, None, 0, P, 8, P, 8, P, 1, 4, 8, P, P, P, P, 1 << 30, None]
    for at, bad, status in ((0, None, INVALID), (1, 9, INVALID), (2, -1, INVALID), (5, None, INVALID), (6, -1, INVALID), (8, -1, INVALID), (9, None, INVALID),
                            (10, 9, INVALID), (11, 0, INVALID), (12, 0, INVALID), (13, None, INVALID), (14, None, INVALID), (16, None, WORKSPACE),
                            (16, P + 2, WORKSPACE), (17, 3, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_rms_norm_q8_backward(*args) == status, (at, bad)


def test_matmul_refuses(lib):
    size = ctypes.c_size_t()
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1 << 31, 1, 1)):
        assert lib.geo_sc_matmul_q8_workspace_size(P, 4096, P, 4096, *sizes, ctypes.byref(size)) == INVALID
        assert lib.geo_sc_matmul_q8_backward_workspace_size(*sizes, 0, 1, 1, ctypes.byref(size)) == INVALID
    # few workgroups and a long inner dimension: cut, with partial sums
    assert lib.geo_sc_matmul_q8_workspace_size(P, 65536, P, 65536, 100, 130, 65536, ctypes.byref(size)) == 0 and size.value >= 2 * 100 * 130 * 4
    assert lib.geo_sc_matmul_q8_workspace_size(P, -1, P, 4096, 100, 130, 4096, ctypes.byref(size)) == INVALID
    # rows at odd addresses are laid out anew, but not for few rows
    cut = size.value
    assert lib.geo_sc_matmul_q8_workspace_size(P, 65537, P, 65536, 100, 130, 65536, ctypes.byref(size)) == 0 and size.value >= cut + 100 * 65536
    assert lib.geo_sc_matmul_q8_workspace_size(P, 65536, P + 1, 65536, 100, 130, 65536, ctypes.byref(size)) == 0 and size.value >= cut + 130 * 65536
    assert lib.geo_sc_matmul_q8_workspace_size(P, 4095, P, 4095, 3, 4096, 4095, ctypes.byref(size)) == 0 and size.value == 0
    good = [P, 4096, P, P, 4096, P, 100, 130, 65536, P, 1, P, 1 << 30, None]
    for at, bad, status in ((0, None, INVALID), (1, -1, INVALID), (2, None, INVALID), (3, None, INVALID), (4, -1, INVALID), (5, None, INVALID),
                            (6, 0, INVALID), (7, 0, INVALID), (8, 131072, INVALID), (9, None, INVALID), (10, 4, INVALID),
                            (11, None, WORKSPACE), (11, P + 4, WORKSPACE), (12, 100, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_matmul_q8(*args) == status, (at, bad)
    good = [P, 1, 130, P, 4096, P, P, 4096, P, 100, 130, 4096, P, 1, P, 1, P, 1 << 40, None]
    for at, bad, status in ((0, None, INVALID), (1, 5, INVALID), (2, -1, INVALID), (3, None, INVALID), (5, None, INVALID), (6, None, INVALID),
                            (8, None, INVALID), (9, 0, INVALID), (10, 131072, INVALID), (13, 5, INVALID), (15, 5, INVALID),
                            (16, None, WORKSPACE), (16, P + 8, WORKSPACE), (17, 100, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_matmul_q8_backward(*args) == status, (at, bad)


def test_distill_refuses(lib):
    size = ctypes.c_size_t()
    assert lib.geo_sc_distill_topk_workspace_size(5, 100003, ctypes.byref(size)) == 0 and size.value > 20
    assert lib.geo_sc_distill_topk_workspace_size(0, 10, ctypes.byref(size)) == INVALID
    good = [P, 1, 10, P, 1, P, 4, 5, 10, 3, 1.0, 2, P, P, P, 1 << 20, None]
    for at, bad, status in ((0, None, INVALID), (1, 3, INVALID), (2, -1, INVALID), (3, None, INVALID), (4, 3, INVALID), (5, None, INVALID), (6, 2, INVALID),
                            (7, 0, INVALID), (8, 0, INVALID), (9, 0, INVALID), (9, 4097, INVALID), (10, 0.0, INVALID), (10, float("nan"), INVALID),
                            (11, 3, INVALID), (12, None, INVALID), (13, None, INVALID), (14, None, WORKSPACE), (15, 3, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_distill_topk(*args) == status, (at, bad)
    good = [P, 2, P, 1, 10, P, 1, P, 4, 5, 10, 3, 1.0, P, P, None]
    for at, bad in ((0, None), (1, 3), (2, None), (3, 3), (4, -1), (5, None), (6, 3), (7, None), (8, 2), (9, 0), (10, 0), (11, 4097), (12, -1.0), (13, None), (14, None)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_distill_topk_backward(*args) == INVALID, (at, bad)


def test_host_tensors_are_refused():
    from geo_amd import utils_functional as uf
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    q, s = torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: uf.quantize_rows(x), lambda: uf.rms_norm_q8(x, w[0]), lambda: uf.matmul_q8(q, s, q, s), lambda: uf.linear_q8(x, w),
                 lambda: uf.norm_linear_q8(x, w[0], w), lambda: uf.distill_topk(x, x[:, :1], q[:, :1].int())):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            call()
