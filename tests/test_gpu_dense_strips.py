"""The 8-bit product and its gradients where their last rows and columns are strips of their own, each form that the plan has of them, against
the formulas in 64 bits."""
import pytest
import torch

from tests.test_dense_strips_plan import BACKWARD, FORWARD, backward, forward
from tests.test_gpu_dense import EPS, TYPES, U, close, product64, rand, random_q8, subnormal, uf  # noqa: F401
from tests.test_gpu_dense_epilogue import check, epilogue64
from tests.test_gpu_dense_kernels import aligned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", FORWARD)
def test_product(uf, shape):
    m, n, k = shape
    assert any(forward(*shape)[1:])
    (q, s), (wq, ws) = random_q8(m, k, 1), random_q8(n, k, 2)
    ws = ws / (k ** 0.5 * 40)
    for x, w in ((aligned(q), aligned(wq)), (q, wq)):   # as they lie, and laid out anew
        for i, dtype in enumerate(TYPES):
            want = product64(x, s, w, ws)
            close(uf.matmul_q8(x, s, w, ws, dtype=dtype), want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))
            check(uf, x, s, w, ws, dtype, ("gelu", "silu", "relu")[i], rand(n, dtype=dtype, seed=3), rand(m, n, dtype=dtype, seed=4))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", BACKWARD)
def test_gradients(uf, case, dtype):
    m, n, k, need_dx, need_dw = case
    assert any(backward(*case, TYPES.index(dtype)))
    x, w = rand(m, k, dtype=dtype, seed=6), rand(n, k, dtype=dtype, seed=7, scale=k ** -0.5)
    bias, g = rand(n, dtype=dtype, seed=8), rand(m, n, dtype=dtype, seed=5)
    x.requires_grad_(need_dx)
    w.requires_grad_(need_dw)
    y = uf.linear_q8(x, w, bias=bias, activation="silu")
    grads = torch.autograd.grad(y, [t for t, need in ((x, need_dx), (w, need_dw)) if need], g)
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    _, _, slope, slope_off, _ = epilogue64(product64(q, s, wq, ws), bias, "silu", None, dtype)
    dz, dz_off = g.double() * slope, g.double().abs() * (slope_off + U * slope.abs())
    xr, wr = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    terms = 1 if dtype == torch.bfloat16 else 2
    kept = EPS[torch.float16] ** terms + U
    left_x, left_w = (dz * ws.double()).abs().amax(1, keepdim=True), (dz * s.double()[:, None]).abs().amax(0)[:, None]
    every = [(dz @ wr, dz.abs() @ wr.abs(), dz_off @ wr.abs(), n, left_x * wq.double().abs().sum(0))] if need_dx else []
    if need_dw:
        every.append((dz.t() @ xr, dz.t().abs() @ xr.abs(), dz_off.t() @ xr.abs(), m, left_w * q.double().abs().sum(0)))
    for got, (want, size, off, depth, low) in zip(grads, every):
        close(got, want, EPS[dtype] * want.abs() + (kept + 2 * terms * depth * U) * size + off + 2.0 ** -39 * low + subnormal(dtype))
