"""Which last rows and columns the 8-bit product and its gradients take as strips of their own, for the shapes that the GPU tests run: rows,
columns and both, in tiles of 128 and of 256, of either gradient and of both together, whatever becomes of the table of costs."""
import ctypes

import pytest

# rows x cols x inner, rows at multiples of 16 bytes: tile, last rows, last columns
FORWARD = {
    (4096, 4099, 300): (128, 0, 3), (4100, 4096, 300): (128, 4, 0), (4111, 4160, 300): (128, 15, 64), (4160, 7937, 260): (128, 64, 1),
    (2049, 8204, 270): (128, 1, 12), (7171, 1025, 257): (128, 3, 1), (6912, 2305, 1280): (256, 0, 1), (2305, 6912, 1281): (256, 1, 0),
    (2049, 7683, 1281): (256, 1, 3),
}
# rows x cols x inner, dx wanted, dw wanted: last rows and columns of dx, of dw (whatever the gradient's type)
BACKWARD = {
    (256, 7680, 1027, False, True): (0, 0, 0, 3), (256, 1027, 7680, False, True): (0, 0, 3, 0), (256, 7169, 1025, False, True): (0, 0, 1, 1),
    (7680, 256, 1025, True, False): (0, 1, 0, 0), (1025, 259, 7424, True, False): (1, 0, 0, 0), (1025, 256, 7169, True, False): (1, 1, 0, 0),
    (512, 1088, 5120, True, True): (0, 0, 64, 0), (256, 768, 8256, True, True): (0, 64, 0, 64), (768, 259, 7441, True, True): (0, 17, 3, 17),
    (785, 256, 7936, True, True): (17, 0, 0, 0), (273, 771, 7168, True, True): (17, 0, 3, 0), (771, 256, 7169, True, True): (3, 1, 0, 1),
    (545, 259, 8225, True, True): (33, 33, 3, 33), (4095, 4099, 2047, True, True): (0, 0, 3, 0),
}


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
