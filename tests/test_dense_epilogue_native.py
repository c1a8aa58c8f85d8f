"""The C entry points of the 8-bit product with an epilogue answer bad arguments by a status, before any GPU call; distances around the
matrix instructions of its tile kernels in the built code."""
import ctypes

import pytest
import torch

from tests.test_native_jumps import kernels
from tests.test_native_tiles import violations

INVALID, WORKSPACE = 1, 3
P = 4096   # an address that is never read: every call here ends in its checks


@pytest.fixture(scope="module")
def lib():
    from geo_amd import _native
    return _native.lib()


def epilogue(**changes):
    from geo_amd import _native
    e = _native.Q8Epilogue(struct_bytes=ctypes.sizeof(_native.Q8Epilogue), bias=P, residual=P, slope=P, residual_stride=130, bias_dtype=1, slope_dtype=2, activation=2)
    for k, v in changes.items():
        setattr(e, k, v)
    return ctypes.byref(e)


def test_forward_refuses(lib):
    good = [P, 4096, P, P, 4096, P, 100, 130, 65536, epilogue(), P, 1, P, 1 << 30, None]
    for at, bad, status in ((0, None, INVALID), (1, -1, INVALID), (2, None, INVALID), (3, None, INVALID), (4, -1, INVALID), (5, None, INVALID),
                            (6, 0, INVALID), (7, 0, INVALID), (8, 131072, INVALID), (9, None, INVALID), (10, None, INVALID), (11, 4, INVALID),
                            (12, None, WORKSPACE), (12, P + 4, WORKSPACE), (13, 100, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_matmul_q8_epilogue(*args) == status, (at, bad)
    for bad in (dict(struct_bytes=8), dict(bias_dtype=3), dict(activation=4), dict(activation=-1), dict(residual_stride=-1), dict(slope_dtype=1), dict(slope_dtype=4), dict(slope_dtype=3)):
        args = list(good)
        args[9] = epilogue(**bad)
        assert lib.geo_sc_matmul_q8_epilogue(*args) == INVALID, bad


def test_backward_refuses(lib):
    size, plain = ctypes.c_size_t(), ctypes.c_size_t()
    query = lib.geo_sc_matmul_q8_epilogue_backward_workspace_size
    for sizes in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1 << 31, 1, 1)):
        assert query(*sizes, 0, 1, 1, 1, ctypes.byref(size)) == INVALID
    assert query(100, 130, 4096, 3, 1, 1, 1, ctypes.byref(size)) == INVALID and query(100, 130, 4096, 1, 1, 1, 1, None) == INVALID
    assert query(100, 130, 4096, 1, 1, 1, 0, ctypes.byref(size)) == 0
    assert lib.geo_sc_matmul_q8_backward_workspace_size(100, 130, 4096, 1, 1, 1, ctypes.byref(plain)) == 0 and size.value == plain.value
    assert query(100, 130, 4096, 1, 1, 1, 1, ctypes.byref(size)) == 0 and size.value > plain.value
    assert query(100, 130, 4096, 1, 0, 0, 1, ctypes.byref(size)) == 0 and size.value >= 130 * 4
    good = [P, 1, 130, P, 2, P, 4096, P, P, 4096, P, 100, 130, 4096, P, 1, P, 1, P, 1, P, 1 << 40, None]
    for at, bad, status in ((0, None, INVALID), (1, 5, INVALID), (2, -1, INVALID), (2, 7, INVALID), (4, 4, INVALID), (4, 1, INVALID), (5, None, INVALID), (7, None, INVALID),
                            (8, None, INVALID), (10, None, INVALID), (11, 0, INVALID), (12, 0, INVALID), (13, 131072, INVALID), (15, 5, INVALID),
                            (17, 5, INVALID), (19, 5, INVALID), (20, None, WORKSPACE), (20, P + 8, WORKSPACE), (21, 100, WORKSPACE)):
        args = list(good)
        args[at] = bad
        assert lib.geo_sc_matmul_q8_epilogue_backward(*args) == status, (at, bad)
    args = list(good)
    args[14] = args[16] = args[18] = None   # no gradient is wanted: nothing to do
    assert lib.geo_sc_matmul_q8_epilogue_backward(*args) == 0


def test_host_tensors_are_refused():
    from geo_amd import utils_functional as uf
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    q, s = torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: uf.matmul_q8(q, s, q, s, activation="relu"), lambda: uf.linear_q8(x, w, bias=w[:, 0]),
                 lambda: uf.norm_linear_q8(x, w[0], w, activation="silu")):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            call()
    for call in (lambda: uf.matmul_q8(q, s, q, s, activation="tanh"), lambda: uf.linear_q8(x, w, activation="tanh"),
                 lambda: uf.norm_linear_q8(x, w[0], w, activation="tanh")):
        with pytest.raises(RuntimeError, match="activation must be"):
            call()


def test_distances_around_the_products_of_the_tile_kernels(tmp_path):
    from geo_amd import _native
    found = {name: code for name, code in kernels(_native.lib_path(), tmp_path).items() if "k_tiles_epilogueI" in name and code}
    assert len(found) == 3   # three tiles
    for name, code in found.items():
        products, bad = violations(code)
        assert products >= 8, name
        assert not bad, (name, [(code[i], code[j]) for i, j in bad[:3]])


def test_teacher_pickled_before_its_layers_had_activations():
    """the relu was the network's own then"""
    import copy
    from geo_amd import network
    net = network.PatchMLP_q8(width=16, hidden=32, depth=2)
    del net.__dict__["gated"]
    for layer in (*net.up, *net.down, net.head, net.embed):
        del layer.__dict__["activation"]
        del layer._parameters["bias"]
    again = copy.deepcopy(net)
    assert not again.gated and [up.activation for up in again.up] == ["relu", "relu"]
    assert all(layer.activation is None and layer.bias is None for layer in (*again.down, again.head, again.embed))
