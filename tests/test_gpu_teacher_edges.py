"""The 8-bit teacher at the ends of its sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_blocks_and_no_images():
    from geo_amd import network
    torch.manual_seed(0)
    x = torch.rand(3, 3, 8, 8, generator=torch.Generator().manual_seed(1)).cuda()
    for depth in (0, 1):
        net = network.PatchMLP_q8(width=32, hidden=64, depth=depth).cuda()
        y = net(x)
        y.square().sum().backward()
        assert y.shape == (3, 10) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
        assert net(x[:0]).shape == (0, 10)
