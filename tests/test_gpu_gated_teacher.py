"""Every block of a gated teacher is normed and gated behind, the last one too."""
import copy

import pytest
import torch

from tests.test_gpu_dense import uf  # noqa: F401

pytestmark = pytest.mark.gpu


def teacher(depth, **more):
    from geo_amd import network
    torch.manual_seed(depth)
    net = network.PatchMLP_q8(width=64, hidden=96, depth=depth, activation="gelu", bias=True, gated=True, **more).cuda()
    with torch.no_grad():
        for name, p in net.named_parameters():
            if "gate" in name or "gain" in name or "scale" in name or "bias" in name:
                p.add_(torch.randn_like(p) * 0.3)
    return net


@pytest.mark.parametrize("depth", [1, 3])
def test_every_block_has_a_gate(uf, depth):
    net = teacher(depth)
    gates = [p for name, p in net.named_parameters() if name.endswith(".gate")]
    assert len(gates) == depth
    x = torch.rand(3, 3, 32, 32).cuda()
    with torch.no_grad():
        want = net(x)
        for gate in gates:   # the block adds nothing to the stream
            kept = gate.clone()
            gate.zero_()
            assert not torch.equal(net(x), want)
            gate.copy_(kept)
        # all closed: what the blocks compute is without effect
        for gate in gates:
            gate.zero_()
        closed = net(x)
        for layer in net.down:
            layer.weight.mul_(-1.5)
        assert torch.equal(net(x), closed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_served_as_trained(uf, dtype):
    net = teacher(2).to(dtype)
    x = torch.rand(5, 3, 32, 32).cuda().to(dtype)
    logits = net(x)
    logits.float().square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and (p.grad != 0).any() for p in net.parameters())
    net.prepare()
    with torch.no_grad():
        assert torch.equal(net(x), logits)


def test_teachers_saved_when_the_last_block_was_not_gated(uf):
    """keep their results: as whole modules and as dicts of tensors"""
    from geo_amd import network, utils_class
    old = teacher(2)
    old.head = utils_class.NormLinear_Q8(64, 10).cuda()   # as it was
    x = torch.rand(3, 3, 32, 32).cuda()
    with torch.no_grad():
        y, total = old.embed(x.unfold(2, 4, 4).unfold(3, 4, 4).permute(0, 2, 3, 1, 4, 5).reshape(3, -1, 48)), None
        for up, down in zip(old.up, old.down):
            wide, total = up(y, total)
            y = down(wide)
        want, _ = old.head((total + y).mean(1))
        assert torch.equal(copy.deepcopy(old)(x), want)
        new = teacher(2)
        assert not new.load_state_dict(old.state_dict()).missing_keys
        assert torch.equal(new(x), want)
        # and inside another module
        outer = torch.nn.Sequential(teacher(2))
        outer.load_state_dict({"0." + k: v for k, v in old.state_dict().items()})
        assert torch.equal(outer(x), want)
        # a dict of today's goes into today's
        now = network.PatchMLP_q8(width=64, hidden=96, depth=2, activation="gelu", bias=True, gated=True).cuda()
        now.load_state_dict(teacher(2).state_dict())
        assert torch.equal(now(x), teacher(2)(x))
