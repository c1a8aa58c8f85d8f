"""Steps counted on the GPU are those of each parameter: one without a gradient makes none, as where they are counted on the host."""
import pytest
import torch

from tests.test_gpu_adamw import graph_of

pytestmark = pytest.mark.gpu


def parameters(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, generator=g).cuda().requires_grad_(True) for n in (300, 17, 1000)]


def give(params, which, seed):
    g = torch.Generator().manual_seed(seed)
    for i, p in enumerate(params):
        one = torch.randn(p.shape, generator=g).cuda()
        p.grad = one if i in which else None


# which parameters have a gradient in each step
PATTERNS = [[(0, 1, 2), (0,), (0, 1, 2), (1, 2), (0, 1, 2)], [(0, 1), (0, 1, 2), (2,), (0, 2), (0, 1, 2)], [(0, 1, 2), (), (1,), (1,), (0, 1, 2)]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pattern", PATTERNS, ids=str)
def test_as_on_the_host(pattern, bits):
    from geo_amd import network
    sides = []
    for capturable in (True, False):
        p = parameters()
        opt = network.AdamW(p, lr=0.05, weight_decay=0.1, capturable=capturable, state_bits=bits)
        for k, which in enumerate(pattern):
            give(p, which, k)
            opt.step()
        sides.append((p, [int(opt.state[t]["step"]) for t in p]))
    assert sides[0][1] == sides[1][1] == [sum(i in which for which in pattern) for i in range(3)]
    assert all(torch.equal(a, b) for a, b in zip(sides[0][0], sides[1][0]))


def test_through_a_dict():
    from geo_amd import network
    a, b = parameters(), parameters(1)
    first, second = (network.AdamW(p, lr=0.05, capturable=True) for p in (a, b))
    for k, which in enumerate([(0, 1, 2), (0,)]):
        give(a, which, k)
        first.step()
    second.load_state_dict(first.state_dict())
    with torch.no_grad():
        for x, y in zip(a, b):
            y.copy_(x)
    for k, which in enumerate([(0, 2), (0, 1, 2), (1,)]):
        for p, opt in ((a, first), (b, second)):
            give(p, which, 10 + k)
            opt.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert [int(first.state[p]["step"]) for p in a] == [int(second.state[p]["step"]) for p in b] == [4, 3, 3]


def test_recorded():
    """a recorded step of some of the parameters is refused until a step like it has been made; then it counts theirs alone"""
    from geo_amd import network
    p, q = parameters(), parameters()
    opt, host = network.AdamW(p, lr=0.05, capturable=True), network.AdamW(q, lr=0.05)
    for params, o in ((p, opt), (q, host)):
        give(params, (0, 1, 2), 0)
        o.step()
        give(params, (0, 2), 1)
    with pytest.raises(RuntimeError, match="counted together"):
        graph_of(opt.step)
    torch.cuda.synchronize()
    assert [int(opt.state[t]["step"]) for t in p] == [1, 1, 1]
    opt.step()
    host.step()
    graph = graph_of(opt.step)   # (records a step, does not make it)
    for _ in range(3):
        graph.replay()
        host.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p, q))
    assert [int(opt.state[t]["step"]) for t in p] == [int(host.state[t]["step"]) for t in q] == [5, 1, 5]


def test_recorded_training_step_of_a_model_that_is_used_in_part():
    """warm-up steps part the counters, the recorded step has them so, and the state is put back"""
    from geo_amd import network
    torch.manual_seed(3)
    x, y = torch.rand(16, 33).cuda(), torch.randint(5, (16,)).cuda()

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.used, self.other = torch.nn.Linear(33, 5), torch.nn.Linear(33, 5)

        def forward(self, v):
            return self.used(v)

    results = []
    for recorded in (True, False):
        torch.manual_seed(4)
        net = Net().cuda()
        masters, criterion = network.make_param_copies(net), torch.nn.CrossEntropyLoss()
        opt = network.AdamW(masters, lr=1e-2, capturable=True)
        for p in net.parameters():   # a step of all
            p.grad = torch.ones_like(p)
        network.apply_update(net, opt, masters)
        for p in net.parameters():
            p.grad = None
        step = network.GraphedTrainStep(net, criterion, opt, masters, x, y) if recorded else \
            (lambda a, b: network.train_step(net, a.clone(), b, criterion, opt, masters))
        losses = [step(x, y).clone() for _ in range(4)]
        results.append([t.clone() for t in losses + masters + list(net.parameters())] + [opt.state[m]["step"].clone() for m in masters])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert [int(t) for t in results[0][-4:]] == [5, 5, 1, 1]


def test_parting_what_a_graph_counts_together():
    """would leave the graph with a count that is not all of theirs: refused, and nothing done; counted apart before, both have their own"""
    from geo_amd import network
    p, q = parameters(), parameters()
    opt, host = network.AdamW(p, lr=0.05, capturable=True), network.AdamW(q, lr=0.05)

    def both(which, seed):
        for params, o in ((p, opt), (q, host)):
            give(params, which, seed)
            o.step()

    both((0, 1, 2), 0)
    graph_of(opt.step)
    before = [t.clone() for t in p]
    give(p, (0,), 1)
    with pytest.raises(RuntimeError, match="counted together"):
        opt.step()
    assert all(torch.equal(a, b) for a, b in zip(p, before)) and [int(opt.state[t]["step"]) for t in p] == [1, 1, 1]
    both((0, 1, 2), 2)
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    # a dict brings counters that no graph has
    saved = opt.state_dict()
    opt = network.AdamW(p, lr=0.05, capturable=True)
    opt.load_state_dict(saved)
    both((0,), 3)
    for t in p:
        t.grad = torch.ones_like(t)
    every = graph_of(opt.step)
    for t in q:
        t.grad = torch.ones_like(t)
    for k in range(3):
        every.replay()
        host.step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    assert [int(opt.state[t]["step"]) for t in p] == [int(host.state[t]["step"]) for t in q] == [6, 5, 5]
