"""The loss at temperatures far from one: as the formula has it where the temperature is taken, refused where its square is no float."""
import pytest
import torch

from tests.test_gpu_distill import check, inputs, uf  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [0.05, 20.0, 100.0])
def test_far_temperatures(uf, temperature):
    check(uf, *inputs(9, 300, 6, torch.float32), temperature)


@pytest.mark.parametrize("temperature", [1e-22, 1e-10, 1e19])
def test_numbers_at_the_ends(uf, temperature):
    """all logits alike: loss 0 and gradient 0 of columns that teacher and student weigh alike, at any temperature"""
    z = torch.full((3, 4), 2.5, device="cuda", requires_grad=True)
    t, index = torch.full((3, 4), -1.0, device="cuda"), torch.arange(4, device="cuda").expand(3, 4)
    loss = uf.distill_topk(z, t, index, temperature=temperature, reduction="none")
    dz, = torch.autograd.grad(loss.sum(), z)
    # (logarithms and exponentials of four equal parts round to a few 2^-24 at most; the loss takes them times T^2, the gradient times T)
    assert torch.isfinite(loss).all() and (loss.abs() <= 16 * 2.0 ** -24 * temperature ** 2).all()
    assert torch.isfinite(dz).all() and (dz.abs() <= 16 * 2.0 ** -24 * temperature).all()


@pytest.mark.parametrize("temperature", [1e-23, 1e-39, 1e-300, 1e20, float("inf")])
def test_temperatures_that_are_refused(uf, temperature):
    with pytest.raises(RuntimeError, match="temperature"):
        uf.distill_topk(*inputs(2, 10, 3, torch.float32), temperature=temperature)
