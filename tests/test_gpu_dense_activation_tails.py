"""The activations of the product's epilogue over their range, every row of every kernel.

gelu: the series has 2 Q(x) to 1.5e-7 absolute (Abramowitz and Stegun 7.1.26) for all x >= 0, so z Q(|z|) to 0.75e-7 |z|; the exponential, the
reciprocal and some ten fp32 operations around them are allowed 16 U of what they give, which is at most the number's tail for z < 0 and z for
z > 0.  Relative to a negative tail that is much: 0.16 % of gelu(-5).  silu: an exponential of a product (1.5 U of its exponent
besides), a reciprocal and a product."""
import pytest
import torch

from tests.test_gpu_dense import U, uf  # noqa: F401
from tests.test_gpu_dense_epilogue import act64

pytestmark = pytest.mark.gpu

SERIES = 0.75e-7


def through_a_product(uf, z, rows, kind):
    """act(z) for `rows` rows: a product of zeros with z as its bias"""
    n = z.numel()
    q, s = torch.zeros(rows, 16, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda")
    wq, ws = torch.zeros(n, 16, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    return uf.matmul_q8(q, s, wq, ws, bias=z, activation=kind)


@pytest.mark.parametrize("rows", [1, 20, 40, 64, 70, 300, 2100])
@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
def test_rows_agree(uf, kind, rows):
    """numbers from the smallest to the largest, infinities and NaN: a row's values do not depend on where it is"""
    z = torch.cat([torch.linspace(-30, 30, 2001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30, 3e38, -3e38, 88.8, -88.8, -104.0, -200.0]),
                   torch.tensor([float("inf"), -float("inf"), float("nan")])]).cuda()
    y = through_a_product(uf, z, rows, kind)
    assert torch.equal(torch.isnan(y), torch.isnan(y[:1]).expand_as(y))
    assert torch.equal(y.nan_to_num(7.0, 8.0, 9.0), y[:1].nan_to_num(7.0, 8.0, 9.0).expand_as(y))
    n, finite = z.numel(), torch.isfinite(z)
    assert torch.isfinite(y[0][finite]).all() and torch.isnan(y[0, n - 1]) and y[0, n - 3] == float("inf")


@pytest.mark.parametrize("rows", [1, 70])
def test_gelu(uf, rows):
    z = torch.cat([torch.linspace(-14, 14, 40001), -torch.logspace(-30, 1, 3000), torch.logspace(-30, 38, 3000)]).cuda()
    want, slope = act64(z.double(), "gelu")
    y = through_a_product(uf, z, rows, "gelu")[-1].double()
    off = SERIES * z.double().abs() + 16 * U * want.abs() + 2.0 ** -149
    assert ((y - want).abs() <= off).all(), ((y - want).abs() / off).max().item()
    # beyond 5.6 (Q < 1e-8) what is wrong is less than half a step of the number itself, and nothing is left of a tail beyond 14
    large = z > 5.6
    assert ((y - z.double()).abs()[large] <= 2 * U * z.double()[large]).all()
    assert (through_a_product(uf, torch.full((64,), -14.5, device="cuda"), rows, "gelu") <= 0).all()


@pytest.mark.parametrize("rows", [1, 70])
def test_silu(uf, rows):
    z = torch.cat([torch.linspace(-80, 80, 40001), -torch.logspace(-30, 1, 3000), torch.logspace(-30, 38, 3000)]).cuda()
    want, _ = act64(z.double(), "silu")
    y = through_a_product(uf, z, rows, "silu")[-1].double()
    off = (16 * U + 3 * U * z.double().abs().clamp(max=90) * (z < 0)) * want.abs() + 2.0 ** -149
    assert ((y - want).abs() <= off).all(), ((y - want).abs() / off).max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["gelu", "silu"])
def test_slopes(uf, kind, dtype):
    """the gradient of the bias of one row is the upstream gradient times the slope: gelu's to the series' bound and 16 U of its parts; kept
    with half a step of fp16 beside bfloat16, of fp32 else"""
    z = torch.cat([torch.linspace(-14, 14, 20001), -torch.logspace(-20, 1, 500), torch.logspace(-20, 30, 500)]).cuda().to(dtype)
    bias, x, w = z.clone().requires_grad_(True), torch.zeros(1, 16, dtype=dtype, device="cuda"), torch.zeros(z.numel(), 16, dtype=dtype, device="cuda")
    d, = torch.autograd.grad(uf.linear_q8(x, w, bias=bias, activation=kind), bias, torch.ones(1, z.numel(), dtype=dtype, device="cuda"))
    _, slope = act64(z.double(), kind)
    parts = slope.abs() + (z.double() * torch.exp(-z.double().square() / 2)).abs() if kind == "gelu" else \
        slope.abs() + z.double().abs().clamp(max=90) * torch.sigmoid(-z.double().abs()) * 3
    kept, least = (2.0 ** -11, 2.0 ** -25) if dtype is torch.bfloat16 else (U, 0.0)
    off = (SERIES if kind == "gelu" else 0) + 16 * U * parts + (kept + torch.finfo(dtype).eps / 2) * slope.abs() + least + 2.0 ** -134
    assert ((d.double() - slope).abs() <= off).all(), ((d.double() - slope).abs() / off).max().item()
