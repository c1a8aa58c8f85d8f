"""What comes back to a NaN in front of a relu goes on through the epilogue, as it does behind torch's relu: the same bits."""
import pytest
import torch

from tests.test_gpu_dense import TYPES, rand, uf  # noqa: F401

pytestmark = pytest.mark.gpu


# few rows, tiles of few stages, tiles of the load ring, an inner dimension that is cut
@pytest.mark.parametrize("shape", [(5, 77, 40), (40, 100, 4160), (70, 130, 100), (300, 257, 700), (130, 300, 9000)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["bias", "row", "gradient"])
def test_gradient_of_a_nan(uf, dtype, shape, where):
    m, n, k = shape
    x, w, bias = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5), rand(n, dtype=dtype, seed=3)
    g = rand(m, n, dtype=dtype, seed=4)
    if where == "bias":
        bias[[0, n // 2, n - 1]] = float("nan")
    elif where == "row":
        x[m // 2, 3] = float("nan")
    else:   # one that meets a NaN, one that meets numbers
        bias[n // 2] = float("nan")
        g[1, n // 2] = float("nan")
        g[2] = float("nan")
    for with_bias in (True, False) if where == "row" else (True,):
        leaves = [t.clone().requires_grad_(True) for t in ((x, w, bias) if with_bias else (x, w))]
        y = uf.linear_q8(*leaves, activation="relu")
        plain = torch.relu(uf.linear_q8(*leaves))
        assert torch.isnan(y).any() and torch.equal(torch.isnan(y), torch.isnan(plain))
        for got, want in zip(torch.autograd.grad(y, leaves, g), torch.autograd.grad(plain, leaves, g)):
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5))
    if where == "bias":   # the bias's gradient is there, and is the sum
        d = torch.autograd.grad(uf.linear_q8(*leaves, activation="relu"), leaves[2], g)[0]
        total = g.double().sum(0)[[0, n // 2, n - 1]]
        off = torch.finfo(dtype).eps / 2 * total.abs() + m * 2.0 ** -24 * g.double().abs().sum(0)[[0, n // 2, n - 1]]
        assert ((d[[0, n // 2, n - 1]].double() - total).abs() <= off + 2.0 ** -25).all()
