"""Which last rows and columns the 8-bit product and its gradients take as strips of their own, for the shapes that the GPU tests run: rows,
columns and both, in tiles of 128 and of 256, of either gradient and of both together, whatever becomes of the table of costs."""
import ctypes

import pytest

# rows x cols x inner, rows at multiples of 16 bytes: tile, last rows, last columns
FORWARD = {
    (5120, 1537, 512): (128, 0, 1), (1297, 6144, 515): (128, 17, 0), (6912, 2305, 1280): (256, 0, 1), (2305, 6912, 1281): (256, 1, 0),
    (2049, 7683, 1281): (256, 1, 3), (4095, 4099, 2047): (256, 0, 3),
}
# rows x cols x inner, dx wanted, dw wanted: last rows and columns of dx, of dw (whatever the gradient's type)
BACKWARD = {
    (256, 6144, 1313, False, True): (0, 0, 0, 33), (256, 1537, 5376, False, True): (0, 0, 1, 0), (768, 3075, 5123, False, True): (0, 0, 3, 3),
    (7680, 256, 1025, True, False): (0, 1, 0, 0), (1025, 259, 7424, True, False): (1, 0, 0, 0), (6147, 768, 2561, True, False): (3, 1, 0, 0),
    (512, 1088, 5120, True, True): (0, 0, 64, 0), (768, 1280, 8195, True, True): (0, 3, 0, 3), (1536, 1539, 5121, True, True): (0, 1, 3, 1),
    (771, 256, 8192, True, True): (3, 0, 0, 0), (832, 1025, 8192, True, True): (64, 0, 1, 0), (1539, 1536, 4928, True, True): (3, 64, 0, 64),
    (4095, 4099, 2047, True, True): (0, 0, 3, 0),
}
# strips that would save a round and cost more: forward, and gradients of any type (measured up to 1.7 times as slow with them)
NOT_WORTH = [(4096, 4099, 300), (4111, 4160, 300), (4160, 7937, 260), (2049, 8204, 270), (2100, 15619, 404), (1326, 6276, 1042), (5558, 1410, 638)]
GRADIENTS_NOT_WORTH = [(1071, 2974, 1955), (545, 259, 8225), (1032, 3628, 1829), (445, 1834, 3767), (2475, 555, 5141), (339, 9938, 5675)]


def forward(rows, cols, inner, x=4096, w=4096, x_stride=None, w_stride=None):
    from geo_amd import _native
    stride = (inner + 15) // 16 * 16
    x_stride, w_stride = x_stride or stride, w_stride or stride
    plan, last = [ctypes.c_int() for _ in range(3)], [ctypes.c_int64(-1) for _ in range(2)]
    assert _native.lib().geo_sc_matmul_q8_plan(x, x_stride, w, w_stride, rows, cols, inner, *[ctypes.byref(v) for v in plan]) == 0
    assert _native.lib().geo_sc_matmul_q8_strips(x, x_stride, w, w_stride, rows, cols, inner, *[ctypes.byref(v) for v in last]) == 0
    return plan[1].value, last[0].value, last[1].value


def backward(rows, cols, inner, dx, dw, grad_type):
    from geo_amd import _native
    last = [ctypes.c_int64(-1) for _ in range(4)]
    assert _native.lib().geo_sc_matmul_q8_backward_strips(rows, cols, inner, grad_type, dx, dw, *[ctypes.byref(v) for v in last]) == 0
    return tuple(v.value for v in last)


@pytest.mark.parametrize("shape", FORWARD)
def test_forward(shape):
    assert forward(*shape) == FORWARD[shape]


@pytest.mark.parametrize("grad_type", [0, 1, 2])
@pytest.mark.parametrize("case", BACKWARD)
def test_backward(case, grad_type):
    assert backward(*case, grad_type) == BACKWARD[case]


@pytest.mark.parametrize("shape", NOT_WORTH)
def test_forward_that_strips_would_slow_down(shape):
    assert forward(*shape) == (128, 0, 0)


@pytest.mark.parametrize("grad_type", [0, 1, 2])
@pytest.mark.parametrize("shape", GRADIENTS_NOT_WORTH)
def test_gradients_that_strips_would_slow_down(shape, grad_type):
    assert backward(*shape, True, True, grad_type) == (0, 0, 0, 0)


def test_none():
    """whole tiles, few rows, a cut inner dimension, tiles of 64, rows that are no round of their own"""
    for shape in ((4096, 4096, 4096), (48, 4099, 16384), (600, 500, 30001), (257, 300, 1111), (1500, 3100, 4000)):
        assert forward(*shape)[1:] == (0, 0), shape
    assert backward(4096, 4096, 4096, True, True, 1) == (0, 0, 0, 0) and backward(300, 257, 77, True, True, 0) == (0, 0, 0, 0)
    assert backward(4095, 4099, 2047, False, False, 1) == (0, 0, 0, 0)


def test_rows_at_other_addresses():
    """are laid out anew, and cut alike"""
    shape = (2049, 7683, 1281)
    assert forward(*shape, x=4097) == forward(*shape, x_stride=1281) == forward(*shape, w=4097, w_stride=1281) == FORWARD[shape]


def test_refusals():
    from geo_amd import _native
    out = [ctypes.byref(ctypes.c_int64()) for _ in range(4)]
    for sizes, strides in (((0, 1, 1), (16, 16)), ((1, 0, 1), (16, 16)), ((1, 1, 0), (16, 16)), ((1, 1, 131072), (16, 16)), ((1, 1, 1), (-1, 16)), ((1, 1, 1), (16, -1))):
        assert _native.lib().geo_sc_matmul_q8_strips(4096, strides[0], 4096, strides[1], *sizes, *out[:2]) == 1
    for i in range(2):
        assert _native.lib().geo_sc_matmul_q8_strips(4096, 16, 4096, 16, 1, 1, 1, *[None if i == k else out[k] for k in range(2)]) == 1
    for i in range(4):
        assert _native.lib().geo_sc_matmul_q8_backward_strips(1, 1, 1, 0, 1, 1, *[None if i == k else out[k] for k in range(4)]) == 1
    assert _native.lib().geo_sc_matmul_q8_backward_strips(1, 1, 1, 3, 1, 1, *out) == 1
    assert _native.lib().geo_sc_matmul_q8_backward_strips(0, 1, 1, 0, 1, 1, *out) == 1
