"""Gradients of a layer with more output columns than an exact integer sum could have terms: the input's gradient sums over them in fp32."""
import pytest
import torch

from tests.test_gpu_dense import EPS, U, close, product64, rand, subnormal, uf  # noqa: F401

pytestmark = pytest.mark.gpu


def check(uf, x, w, g, dx, dw):
    """as test_linear has it: fp16 terms of the scaled gradient, fp32 sums of all terms"""
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    xr, wr, g64 = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], g.double()
    dtype, terms = x.dtype, 1 if g.dtype == torch.bfloat16 else 2
    kept = EPS[torch.float16] ** terms + U
    left_x, left_w = (g64 * ws.double()).abs().amax(1, keepdim=True), (g64 * s.double()[:, None]).abs().amax(0)[:, None]
    for got, want, size, depth, low in ((dx, g64 @ wr, g64.abs() @ wr.abs(), g.shape[1], left_x * wq.double().abs().sum(0)),
                                        (dw, g64.t() @ xr, g64.t().abs() @ xr.abs(), g.shape[0], left_w * q.double().abs().sum(0))):
        close(got, want, EPS[dtype] * want.abs() + (kept + 2 * terms * depth * U) * size + 2.0 ** -39 * low + subnormal(dtype))
    return product64(q, s, wq, ws)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 140000, 8), (70, 131072, 40), (129, 151936, 33)])
def test_linear_with_many_columns(uf, dtype, shape):
    m, n, k = shape
    x, w, g = rand(m, k, dtype=dtype, seed=1).requires_grad_(True), rand(n, k, dtype=dtype, seed=2).requires_grad_(True), rand(m, n, dtype=dtype, seed=3, scale=1e-2)
    y = uf.linear_q8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    want = check(uf, x, w, g, dx, dw)
    close(y, want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))


def test_gradients_with_rows_that_overlap_or_are_one(uf):
    x, w = rand(9, 24, seed=1).requires_grad_(True), rand(30, 24, seed=2).requires_grad_(True)
    base = rand(400, seed=3)
    for g in (base.as_strided((9, 30), (7, 1)), base.as_strided((9, 30), (0, 1)), base.as_strided((9, 30), (1, 9)), base[:1].expand(9, 30)):
        got = torch.autograd.grad(uf.linear_q8(x, w), (x, w), g)
        want = torch.autograd.grad(uf.linear_q8(x, w), (x, w), g.contiguous().clone())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_columns_at_all(uf, dtype):
    """sums of nothing"""
    x, w = rand(5, 24, dtype=dtype, seed=1).requires_grad_(True), torch.empty(0, 24, dtype=dtype, device="cuda", requires_grad=True)
    gain = torch.ones(24, dtype=dtype, device="cuda", requires_grad=True)
    y = uf.linear_q8(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (5, 0) and dx.shape == (5, 24) and dx.dtype == dtype and (dx == 0).all() and dw.shape == (0, 24)
    y, total = uf.norm_linear_q8(x, gain, w, residual=x.detach())
    h = rand(5, 24, dtype=dtype, seed=2)
    dx, dgain, dw = torch.autograd.grad((y, total), (x, gain, w), (torch.empty_like(y), h))
    assert torch.equal(dx, h) and (dgain == 0).all() and dw.shape == (0, 24)
