"""A refusal names the operators that it is about."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_gated_norm():
    from geo_amd import utils_functional as uf
    x, w = torch.ones(4, 40, device="cuda"), torch.ones(40, device="cuda")
    with pytest.raises(RuntimeError, match="gated norm.*cannot be traced"):
        torch.jit.trace(lambda t: uf.gated_norm(t, t, w)[0], (x,))
    y = x.clone().requires_grad_(True)
    for out in uf.gated_norm(y, x, w):
        d, = torch.autograd.grad(out.sum(), y, create_graph=True)
        with pytest.raises(RuntimeError, match="gated norm.*once only"):
            torch.autograd.grad(d.sum(), y)
