"""Rows of any magnitude through the norm with 8-bit output: where squares, or products with the weight, pass fp32's range the result
is still the formula's, forward and backward."""
import pytest
import torch

from tests.test_gpu_dense import EPS, U, check_rows, close, norm64, norm_gradients64, rand, subnormal, uf  # noqa: F401

pytestmark = pytest.mark.gpu

# within a block's registers: one wave per row, several; two kernels for longer rows
COLS = [5, 64, 513, 4096, 40007]


def rows_of_many_magnitudes(cols, dtype, seed):
    """row r times 2^e: sums of squares beyond the largest float and below the smallest, the type's ends among them"""
    e = torch.tensor([-126, -120, -90, -75, -60, -40, 0, 40, 62, 63, 64, 90, 120, 124])
    x = rand(len(e), cols, seed=seed).clamp(-4, 4).double() * (2.0 ** e.double())[:, None].cuda()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norm_of_rows_of_any_magnitude(uf, dtype, cols, eps):
    x, w = rows_of_many_magnitudes(cols, dtype, 1), (1 + rand(cols, seed=3, scale=0.2)).to(dtype)
    for residual in (None, rows_of_many_magnitudes(cols, dtype, 2) / 4):
        q, scale, total, values = uf.rms_norm_q8(x, w, residual=residual, eps=eps, values=torch.float32)
        t, r, n = norm64(x, w, residual, eps)
        # as of ordinary rows; x + residual below 2^-126 rounds to steps of 2^-149, which r lifts
        slack = (cols / 64 + 64) * U
        check_rows(q, scale, n, slack=slack + (2.0 ** -149 / t.abs().amax(-1)).max().item())
        close(values, q.double() * scale.double().unsqueeze(-1), 2 * U * values.double().abs() + 2.0 ** -149)
        assert torch.isfinite(scale).all()


@pytest.mark.parametrize("cols", [64, 4096])
def test_norm_with_a_weight_of_another_magnitude(uf, cols):
    """t w alone passes the range, t r w does not"""
    x, w = rand(6, cols, seed=1), rand(cols, seed=2)
    for up, weight in ((2.0 ** 60, 2.0 ** 80), (2.0 ** -70, 2.0 ** -75), (2.0 ** 100, 2.0 ** -20)):
        q, scale, _, _ = uf.rms_norm_q8(x * up, w * weight, eps=0.0)
        check_rows(q, scale, norm64(x * up, w * weight, None, 0.0)[2], slack=(cols / 64 + 64) * U)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 513, 4096, 20011])
def test_norm_backward_of_rows_of_any_magnitude(uf, dtype, cols):
    x = rows_of_many_magnitudes(cols, dtype, 1)[4:-1].contiguous()   # (r itself is a float of full precision)
    rows = x.shape[0]
    x, w = x.requires_grad_(True), (1 + rand(cols, seed=3, scale=0.2)).to(dtype).requires_grad_(True)
    g = rand(rows, cols, seed=4).to(dtype)
    _, _, _, values = uf.rms_norm_q8(x, w, eps=0.0, values=dtype)
    dx, dw = torch.autograd.grad(values, (x, w), g)
    want_x, size_x, want_w, size_w = norm_gradients64(x.detach(), w.detach(), 0.0, g, None)
    close(dx, want_x, EPS[dtype] * want_x.abs() + (cols / 64 + 80) * U * size_x + subnormal(dtype))
    close(dw, want_w, EPS[dtype] * want_w.abs() + (rows / 64 + 80) * U * size_w + subnormal(dtype))


def test_rows_that_are_no_numbers_stay_so(uf):
    for cols in (64, 4096, 40007):
        x, w = rand(6, cols, seed=1) * 2.0 ** 70, torch.ones(cols, device="cuda")
        x[0, 3], x[1, cols - 1], x[2] = float("inf"), float("nan"), 0
        q, scale, _, values = uf.rms_norm_q8(x, w, values=torch.float32)
        assert torch.isnan(scale[:2]).all() and (q[:2] == 0).all() and torch.isnan(values[:2]).all()
        assert scale[2] == 0 and (q[2] == 0).all() and torch.isfinite(scale[2:]).all()
        x[3:] = float("inf")
        w[5] = float("inf")
        assert torch.isnan(uf.rms_norm_q8(x[4:], w)[1]).all()
