"""How the AdamW step goes over its tensors: launches of up to 48, past the caches where what is written passes half of them.  On the host."""
import ctypes

import pytest

INVALID, UNSUPPORTED = 1, 5
F32, BF16, F16 = 0, 1, 2


def plan(sizes, bits=32, param=F32, grad=F32, copy=None, clamped=False, shift=(), struct_bytes=None):
    from geo_amd import _native
    places = dict(param=1 << 20, grad=2 << 20, exp_avg=3 << 20, exp_avg_sq=4 << 20, avg_scale=5 << 20, sq_scale=6 << 20,
                  copy=7 << 20 if copy is not None else None, clamped=8 << 20 if clamped else None)
    for name in shift:
        places[name] += 4
    tensors = (_native.AdamWTensor * max(1, len(sizes)))(*[_native.AdamWTensor(elements=n, **places) for n in sizes])
    o = _native.AdamWOptions(struct_bytes=ctypes.sizeof(_native.AdamWOptions) if struct_bytes is None else struct_bytes, state_bits=bits, lr=1e-3,
                             beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, lo=-1, hi=1, step=1, param_dtype=param, grad_dtype=grad,
                             copy_dtype=copy or 0)
    launches, uncached = ctypes.c_int(-1), ctypes.c_int(-1)
    rc = _native.lib().geo_sc_adamw_plan(len(sizes), tensors, ctypes.byref(o), ctypes.byref(launches), ctypes.byref(uncached))
    return (launches.value, uncached.value) if rc == 0 else rc


HALF = 128 << 20   # bytes


@pytest.mark.parametrize("more,written", [
    (dict(), 12), (dict(copy=BF16), 14), (dict(copy=F32), 16), (dict(clamped=True), 16), (dict(copy=F32, clamped=True), 20),
    (dict(bits=8), 6), (dict(bits=8, clamped=True), 10), (dict(bits=8, param=BF16), 4), (dict(bits=8, param=F16, copy=F16, clamped=True), 10),
    (dict(param=BF16, clamped=True), 14)], ids=str)
def test_what_is_written_counts(more, written):
    """parameters, states, copies and clamped copies"""
    least = -(-HALF // written)
    assert plan([least], **more) == (1, 1) and plan([least - 1], **more) == (1, 0)
    assert plan([least // 3, least // 3, least - 2 * (least // 3)], **more) == (1, 1)


def test_places():
    """what is loaded starts at a multiple of 16 bytes; codes, scales and copies may start anywhere"""
    n = HALF // 4
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert plan([n], shift=[name]) == (1, 0)
    for name in ("exp_avg", "exp_avg_sq", "avg_scale", "sq_scale", "copy", "clamped"):
        assert plan([n], bits=8, copy=F32, clamped=True, shift=[name]) == (1, 1)


def test_launches():
    assert plan([]) == (0, 0) and plan([0, 0]) == (0, 0)
    for count, launches in ((1, 1), (48, 1), (49, 2), (96, 2), (97, 3)):
        assert plan([100] * count) == (launches, 0)
    assert plan([100, 0] * 48) == (1, 0)          # empty ones are left out
    most = 2048 * (0xffffffff // 256)             # elements of one launch's threads
    assert plan([most]) == (1, 1) and plan([most, 1]) == (2, 1) and plan([1, most]) == (2, 1)


def test_refusals():
    from geo_amd import _native
    assert plan([-1]) == INVALID and plan([1], bits=16) == INVALID and plan([1], struct_bytes=8) == INVALID
    assert plan([1 << 50]) == UNSUPPORTED
    one = ctypes.c_int()
    o = _native.AdamWOptions(struct_bytes=ctypes.sizeof(_native.AdamWOptions), state_bits=32, lo=-1, hi=1, step=1)
    query = _native.lib().geo_sc_adamw_plan
    assert query(0, None, ctypes.byref(o), None, ctypes.byref(one)) == INVALID
    assert query(0, None, ctypes.byref(o), ctypes.byref(one), None) == INVALID
    assert query(1, None, ctypes.byref(o), ctypes.byref(one), ctypes.byref(one)) == INVALID
    assert query(0, None, None, ctypes.byref(one), ctypes.byref(one)) == INVALID
