"""The dense layers as modules, the 8-bit teacher and the command that distils an SC network from it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def images(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.rand((n, 3, 32, 32), generator=g).cuda(), torch.randint(10, (n,), generator=g).cuda()


def test_prepared_layers_give_the_values_of_unprepared_ones():
    from geo_amd import network
    torch.manual_seed(0)
    net = network.PatchMLP_q8(width=64, hidden=160, depth=2).cuda().eval()
    x, _ = images(9)
    with torch.no_grad():
        before = net(x)
        net.prepare()
        assert torch.equal(net(x), before)
        net.embed.weight.mul_(2)
        assert torch.equal(net(x), before)          # what was prepared stays until it is dropped
        net.train()
        net.eval()
        assert not torch.equal(net(x), before)
        net.prepare()
        net.load_state_dict(net.state_dict())
        assert net.embed._q8 is None and net.head._q8 is None
    with pytest.raises(ValueError, match="patches"):
        net(x[:, :, :30])


def rounded(x):
    """rows in 8 bits in the tensor's own precision, the gradient straight through"""
    a = x.detach().abs().amax(-1, keepdim=True)
    return x + ((x.detach() * (127 / a)).round() * a / 127 - x.detach())


def plain_teacher(net, params, images):
    """PatchMLP_q8.forward from elementary operations on the parameters in 64 bits"""
    def norm(x, gain):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain

    n, p = images.shape[0], net.patch
    rows = images.unfold(2, p, p).unfold(3, p, p).permute(0, 2, 3, 1, 4, 5).reshape(n, -1, 3 * p * p)
    y, total = rounded(rows) @ rounded(params["embed.weight"]).t(), 0.0
    for i in range(len(net.up)):
        total = total + y
        wide = rounded(norm(total, params[f"up.{i}.gain"])) @ rounded(params[f"up.{i}.weight"]).t()
        y = rounded(wide.relu()) @ rounded(params[f"down.{i}.weight"]).t()
    return rounded(norm((total + y).mean(1), params["head.gain"])) @ rounded(params["head.weight"]).t()


def test_teacher_learns_and_its_gradients_are_those_of_its_products():
    """All gradients against the network from elementary operations in 64 bits: numbers next to a half step round to
    different sides there, and a step in one layer moves some more in the next, which the bound of 2 % leaves room for.  The loss
    falls; a layer's gradient is the one of its rounded operands."""
    from geo_amd import network
    from geo_amd import utils_functional as uf
    torch.manual_seed(0)
    net = network.PatchMLP_q8(width=64, hidden=128, depth=2).cuda()
    x, t = images(64)
    params = {k: v.detach().double().requires_grad_(True) for k, v in net.named_parameters()}
    want = torch.nn.functional.cross_entropy(plain_teacher(net, params, x.double()), t)
    want.backward()
    loss = torch.nn.functional.cross_entropy(net(x), t)
    loss.backward()
    assert abs(loss.item() - want.item()) <= 2e-2 * want.item()
    for name, v in net.named_parameters():
        assert (v.grad.double() - params[name].grad).norm() <= 2e-2 * params[name].grad.norm(), name
    optimizer = torch.optim.Adam(net.parameters(), lr=2e-3)
    for _ in range(30):
        last = torch.nn.functional.cross_entropy(net(x), t)
        optimizer.zero_grad()
        last.backward()
        optimizer.step()
    assert last.item() < loss.item()
    layer, rows = net.down[0], torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).cuda()
    g = torch.randn(50, 64, generator=torch.Generator().manual_seed(2)).cuda()
    layer.weight.grad = None
    layer(rows).backward(g)
    q, s, _ = uf.quantize_rows(rows)
    want = g.double().t() @ (q.double() * s.double()[:, None])
    assert (layer.weight.grad.double() - want).abs().max() <= 1e-5 * want.abs().max()


def test_top_logits_are_ordered_and_ties_take_the_lowest_column():
    from geo_amd import main_distill
    logits = torch.tensor([[1.0, 3.0, 3.0, 0.0, 3.0], [5.0, 4.0, 3.0, 2.0, 1.0]]).cuda()
    values, columns = main_distill.top_logits(lambda x: x, logits, 3)
    assert columns.tolist() == [[1, 2, 4], [0, 1, 2]] and values.tolist() == [[3, 3, 3], [5, 4, 3]]


def test_distill_step_follows_the_loss_of_its_formula():
    """the step's loss against log_softmax in 64 bits on the student's own logits; the student moves"""
    from geo_amd import main_conv, main_distill, network
    torch.manual_seed(0)
    teacher = network.PatchMLP_q8(width=64, hidden=128, depth=1).cuda().eval()
    teacher.prepare()
    student = main_conv.build_model(main_distill.build_parser().parse_args(["--err", "5555"])).cuda().train()
    copies = network.make_param_copies(student)
    optimizer = torch.optim.Adam(copies, lr=2e-3)
    x, t = images(64)
    seen = []
    handle = student.register_forward_hook(lambda m, i, o: seen.append(o.detach().double()))
    before = [c.detach().clone() for c in copies]
    loss = main_distill.distill_step(student, teacher, x, t, optimizer, copies, top=4, temperature=3.0, alpha=0.7)
    handle.remove()
    with torch.no_grad():
        values, columns = teacher(x).double().topk(4, dim=1)
    log_p, log_q = torch.log_softmax(values / 3, 1), torch.log_softmax(seen[0] / 3, 1).gather(1, columns)
    want = 0.7 * 9 * (log_p.exp() * (log_p - log_q)).sum(1).mean() + 0.3 * torch.nn.functional.cross_entropy(seen[0], t)
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    assert any(not torch.equal(a, b) for a, b in zip(before, copies))


def test_command_runs():
    from geo_amd import main_distill
    out = main_distill.main(["--dataset", "SYNTHETIC", "--err", "5555", "--batch", "64", "--synthetic_size", "256", "--epochs", "2",
                             "--teacher_epochs", "3"])
    assert len(out["history"]) == 2 and len(out["teacher_losses"]) == 3
    assert out["teacher_losses"][-1] < out["teacher_losses"][0]
    assert all(0 <= h["val_prec1"] <= 100 and h["loss"] == h["loss"] for h in out["history"])
