"""The AdamW step on many tensors against its formulas, in 32-bit operations one by one (the same bits) and in 64 bits; states of 8 bits;
graphs, streams and refusals; the optimiser in the framework's training step."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
LR, BETAS, ADAM_EPS, DECAY = 3e-3, (0.9, 0.99), 1e-8, 0.1
# one element, parts of a chunk, a block's and a workgroup's edges; more tensors than a launch takes
SIZES = [1, 7, 8, 9, 255, 256, 257, 511, 2047, 2048, 2049, 5000, 0, 70001] + [3 + 5 * i for i in range(50)]


@pytest.fixture(scope="module")
def uf():
    assert torch.cuda.is_available(), "these tests need the GPU"
    from geo_amd import utils_functional as m
    return m


def tensors(seed, scale, dtype=torch.float32, sizes=SIZES):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtype).cuda() for n in sizes]


def eight(values):
    """float8 codes and scales of a list of tensors"""
    codes, scales = [], []
    for v in values:
        blocks = torch.nn.functional.pad(v.float(), (0, -v.numel() % 256)).reshape(-1, 256)
        scale = torch.exp2(torch.floor(torch.log2(blocks.abs().amax(1).clamp(min=2.0 ** -100))) - 7)
        codes.append((blocks / scale[:, None]).to(torch.float8_e4m3fn).reshape(-1)[:v.numel()].clone())
        scales.append(scale.to(torch.float8_e8m0fnu))
    return codes, scales


def values(codes, scales):
    """what float8 codes and their scales stand for, in 64 bits"""
    return [c.double() * s.double().repeat_interleave(256)[:c.numel()] for c, s in zip(codes, scales)]


def formula(p, g, m, v, t, scale=1.0, wide=True, lr=LR):
    """(p, m, v) after the step, in 64 bits or in 32-bit operations one by one"""
    kind = torch.float64 if wide else torch.float32
    p, g, m, v = (x.to(kind) for x in (p, g, m, v))
    b1, b2 = BETAS
    g = g * scale
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = p * (1 - lr * DECAY) - (m * (lr / (1 - b1 ** t))) / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + ADAM_EPS)
    return p, m, v


def close(got, want, tolerance):
    got, want = got.double(), want.double()
    bad = (got - want).abs() > tolerance
    assert not bad.any(), (int(bad.sum()), ((got - want).abs() / tolerance)[bad].max().item())


@pytest.mark.parametrize("grad_type", TYPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_states_of_32_bits(uf, dtype, grad_type):
    p, g = tensors(1, 0.1, dtype), tensors(2, 0.5, grad_type)
    m, v = tensors(3, 0.01), [x.square() for x in tensors(4, 0.02)]
    for copy_type in TYPES:
        out = [[x.clone() for x in xs] for xs in (p, m, v)]
        copies = [torch.full_like(x, 7, dtype=copy_type) for x in p]
        clamped = [torch.full_like(x, 7, dtype=torch.float32) if i % 2 else None for i, x in enumerate(p)]
        uf.adamw_step(out[0], g, out[1], out[2], 7, LR, BETAS, ADAM_EPS, DECAY, 1 / 64, copies=copies, clamped=clamped, bounds=(-0.1, 0.05))
        for i in range(len(SIZES)):
            want_p, want_m, want_v = formula(p[i], g[i], m[i], v[i], 7, 1 / 64, wide=False)
            assert torch.equal(out[1][i], want_m) and torch.equal(out[2][i], want_v)
            assert torch.equal(out[0][i], want_p.to(dtype)) and torch.equal(copies[i], want_p.to(copy_type))
            if clamped[i] is not None:
                assert torch.equal(clamped[i], want_p.clamp(-0.1, 0.05))
            # 64 bits: constants, products and sums round once each (U); the quotient's parts 3 + 4 of them, the difference one
            exact_p, exact_m, exact_v = formula(p[i], g[i], m[i], v[i], 7, 1 / 64)
            size_m = 0.9 * m[i].double().abs() + 0.1 * g[i].double().abs() / 64
            close(out[1][i], exact_m, 4 * U * size_m)
            close(out[2][i], exact_v, 6 * U * exact_v)
            update = LR / (1 - 0.9 ** 7) * size_m / (exact_v.sqrt() / math.sqrt(1 - 0.99 ** 7) + ADAM_EPS)
            close(out[0][i], exact_p, 16 * U * update + 3 * U * p[i].double().abs() + EPS[dtype] * exact_p.abs() + 2.0 ** -25)


def test_views_at_odd_places(uf):
    """tensors side by side in flat buffers, at odd elements; what lies between and behind them stays"""
    sizes = [5, 300, 1, 2049, 17]
    for bits in (32, 8):
        flat = [torch.full((4000,), 3.0, device="cuda"), torch.full((4000,), 2.0, device="cuda", dtype=torch.bfloat16)]
        state = [torch.zeros(4000, device="cuda", dtype=torch.float32 if bits == 32 else torch.float8_e4m3fn) for _ in range(2)]
        at, views = 3, []
        for n in sizes:
            views.append(slice(at, at + n))
            at += n + 1
        scales = None if bits == 32 else tuple([torch.zeros((n + 255) // 256, device="cuda", dtype=torch.float8_e8m0fnu) for n in sizes]
                                               for _ in range(2))
        flat[1][::3] = -0.5
        before = flat[0].clone()
        uf.adamw_step(*[[f[s] for s in views] for f in (flat[0], flat[1], *state)], 1, LR, BETAS, ADAM_EPS, DECAY, scales=scales)
        inside = torch.zeros(4000, dtype=torch.bool, device="cuda")
        for s in views:
            inside[s] = True
            want, _, _ = formula(before[s], flat[1][s], torch.zeros_like(before[s]), torch.zeros_like(before[s]), 1, wide=False)
            assert torch.equal(flat[0][s], want)
        assert (flat[0][~inside] == 3).all() and (flat[1][~inside].abs() <= 2).all()
        assert all((s[~inside].float() == 0).all() and (s[inside].float() != 0).all() for s in state)


@pytest.mark.parametrize("dtype", TYPES)
def test_states_of_8_bits(uf, dtype):
    p, g = tensors(1, 0.1, dtype), tensors(2, 0.5)
    (m, ms), (r, rs) = eight(tensors(3, 0.01)), eight([x.abs() + 1e-3 for x in tensors(4, 0.02)])
    lists = [[x.clone() for x in xs] for xs in (p, m, r, ms, rs)]
    uf.adamw_step(lists[0], g, lists[1], lists[2], 5, LR, BETAS, ADAM_EPS, DECAY, scales=(lists[3], lists[4]))
    old = values(m, ms), [x.square() for x in values(r, rs)]
    new = values(lists[1], lists[3]), values(lists[2], lists[4])
    for i, n in enumerate(SIZES):
        # the parameters do not see the rounding of the new states
        want, want_m, want_v = formula(p[i], g[i], old[0][i], old[1][i], 5, wide=False)
        assert torch.equal(lists[0][i], want.to(dtype))
        for got, exact, scale in ((new[0][i], want_m.double(), lists[3][i]), (new[1][i], want_v.sqrt().double(), lists[4][i])):
            if not n:
                continue
            largest = torch.nn.functional.pad(exact.abs(), (0, -n % 256)).reshape(-1, 256).amax(1)
            assert torch.equal(scale.double(), torch.exp2(torch.floor(torch.log2(largest)) - 7))
            # one of the two codes around a number: they are less than an eighth of the power of two below it apart, 2^-9 of the scale
            unit = scale.double().repeat_interleave(256)[:n]
            step = torch.maximum(torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=1e-30))) - 3), unit * 2.0 ** -9)
            assert ((got - exact).abs() < step * (1 + 1e-6)).all()
            assert (got[exact.abs() > step].sign() == exact[exact.abs() > step].sign()).all()
        assert (new[1][i] > 0).all()


def test_rounding_of_8_bits_is_even_over_steps_and_places(uf):
    """m = 0.1 g of constant gradients from zero states: the codes' mean over the steps and over a block is the number itself"""
    n, steps = 256, 512
    g = [torch.full((n,), 1.0, device="cuda")]
    g[0][1:] = 0.6   # times 2^11: 204.8 and 122.88, of codes 16 and 8 apart
    total = torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in range(1, steps + 1):
        m, r = ([torch.zeros(n, device="cuda").to(torch.float8_e4m3fn)] for _ in range(2))
        ms, rs = ([torch.zeros(1, device="cuda", dtype=torch.float8_e8m0fnu)] for _ in range(2))
        uf.adamw_step([torch.zeros(n, device="cuda")], g, m, r, t, LR, BETAS, ADAM_EPS, DECAY, scales=(ms, rs))
        one = values(m, ms)[0]
        total += one
        # of 255 places a fraction of the circle holds its share to within 4 (arcs of 0x9E3779B1 k mod 2^32: at most 3.1 off)
        assert abs(one[1:].mean().item() - 0.06) <= 2.0 ** -8 * 4 / 255 + 1e-8
    # and of 512 steps (0x6A09E667 t: at most 3.2 off)
    step = torch.full((n,), 2.0 ** -8, dtype=torch.float64, device="cuda")
    step[0] = 2.0 ** -7
    assert ((total / steps - 0.1 * g[0].double()).abs() <= step * 4 / steps + 1e-8).all()


def test_8_bit_root_follows_a_gradient_that_changes(uf):
    """three codes' digits and 1 - beta2 = 1/1000: to the nearest, the root would stay; here it reaches the new gradient's to within a code"""
    n, betas = 600, (0.9, 0.999)
    p, (m, ms), (r, rs) = [torch.zeros(n, device="cuda")], eight([torch.zeros(n, device="cuda")]), eight([torch.full((n,), 1.0, device="cuda")])
    g = [torch.full((n,), 3.0, device="cuda")]
    g[0][::2] = -0.3
    for t in range(1000, 8000):
        uf.adamw_step(p, g, m, r, t, 1e-6, betas, ADAM_EPS, 0.0, scales=(ms, rs))
    want = g[0].abs().double()
    # 7000 steps leave e^-7 of the old square: of 1 against 0.09 that is 1 %; a code is up to an eighth of a number
    assert ((values(r, rs)[0] / want - 1).abs() <= 0.125 + 0.02).all()
    assert ((values(m, ms)[0] / g[0].double() - 1).abs() <= 0.125 + 1e-6).all()


def test_numbers_that_are_none(uf):
    for bits in (32, 8):
        n = 1000
        p, g = [torch.ones(n, device="cuda")], [torch.full((n,), 0.5, device="cuda")]
        g[0][300], g[0][301], g[0][700] = float("nan"), float("inf"), -float("inf")
        kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
        state = [[torch.zeros(n, device="cuda", dtype=kind)] for _ in range(2)]
        scales = None if bits == 32 else tuple([torch.zeros(4, device="cuda", dtype=torch.float8_e8m0fnu)] for _ in range(2))
        clamped = [torch.zeros(n, device="cuda")]
        uf.adamw_step(p, g, *state, 1, LR, BETAS, ADAM_EPS, DECAY, scales=scales, clamped=clamped)
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[[300, 301, 700]] = True
        want, m, v = formula(torch.ones(n, device="cuda"), g[0], torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), 1, wide=False)
        assert torch.equal(torch.isnan(p[0]), torch.isnan(want)) and torch.equal(p[0][~bad], want[~bad])
        assert torch.equal(torch.isnan(clamped[0]), torch.isnan(want))
        if bits == 8:
            got_m, got_r = values(state[0], scales[0])[0], values(state[1], scales[1])[0]
            assert torch.equal(torch.isnan(got_m), bad) and torch.equal(torch.isnan(got_r), bad)
            assert ((got_m[~bad] / m[~bad].double() - 1).abs() <= 0.125).all()
        else:
            assert torch.equal(torch.isnan(state[0][0]), torch.isnan(m)) and torch.equal(state[0][0][~bad], m[~bad])


def test_tiny_and_zero_gradients_in_8_bits(uf):
    g = [torch.cat([torch.zeros(256), torch.full((256,), 1e-30), torch.tensor([1.0] + [1e-12] * 255)]).cuda()]
    n = g[0].numel()
    p = [torch.ones(n, device="cuda")]
    state = [[torch.zeros(n, device="cuda").to(torch.float8_e4m3fn)] for _ in range(2)]
    scales = tuple([torch.zeros(3, device="cuda", dtype=torch.float8_e8m0fnu)] for _ in range(2))
    for t in range(1, 4):
        uf.adamw_step(p, g, *state, t, LR, BETAS, ADAM_EPS, 0.0, scales=scales)
        assert torch.isfinite(p[0]).all()
    root = values(state[1], scales[1])[0]
    # zeros stay; squares of 1e-30 are zero in fp32; what is far below its block's largest keeps the smallest code
    assert (root[:512] == 0).all() and (root[512:] > 0).all() and (p[0][:256] == 1).all()


def graph_of(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    return graph


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_two_graphs(uf, bits):
    """two recorded steps of different tensors, replayed in turn between eager work, against eager steps"""
    sets = []
    for seed in (1, 2):
        p, g = tensors(seed, 0.1), tensors(seed + 10, 0.5)
        if bits == 8:
            (m, ms), (r, rs) = eight([x * 0 for x in p]), eight([x * 0 for x in p])
            scales = (ms, rs)
        else:
            m, r, scales = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p], None
        sets.append(dict(p=p, g=g, m=m, r=r, scales=scales))
    clones = copy.deepcopy(sets)
    counts = [torch.zeros(1, dtype=torch.int64, device="cuda") for _ in sets]
    step = lambda s, t: uf.adamw_step(s["p"], s["g"], s["m"], s["r"], t, LR, BETAS, ADAM_EPS, DECAY, scales=s["scales"])   # noqa: E731
    graphs = [graph_of(lambda s=s, c=c: step(s, c)) for s, c in zip(sets, counts)]
    for t in range(1, 5):
        for k, (s, other) in enumerate(zip(sets, clones)):
            for x, y in zip(s["g"], other["g"]):
                x.mul_(0.9)
                y.mul_(0.9)
            graphs[k].replay()
            step(other, t)
            torch.cuda.synchronize()
            assert counts[k].item() == t
            for name in "pmr":
                assert all(torch.equal(x.float(), y.float()) for x, y in zip(s[name], other[name])), (t, k, name)


def test_on_another_stream(uf):
    p, g = tensors(1, 0.1, sizes=[1 << 22]), tensors(2, 0.5, sizes=[1 << 22])
    m, v = [torch.zeros_like(p[0])], [torch.zeros_like(p[0])]
    want, _, _ = formula(p[0], g[0], m[0], v[0], 1, wide=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        uf.adamw_step(p, g, m, v, 1, LR, BETAS, ADAM_EPS, DECAY)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p[0], want)


def test_refusals(uf):
    x = torch.zeros(512, device="cuda")
    y = lambda: torch.zeros(512, device="cuda")   # noqa: E731
    f8, e8 = lambda: y().to(torch.float8_e4m3fn), lambda n=2: torch.zeros(n, device="cuda", dtype=torch.float8_e8m0fnu)   # noqa: E731
    step = lambda *a, **k: uf.adamw_step(*a, 1, LR, **k)   # noqa: E731
    for call, words in (
            (lambda: step([x, x], [y(), y()], [y(), y()], [y(), y()]), "twice"),
            (lambda: step([x], [y()], [x], [y()]), "twice"),
            (lambda: step([x], [y()], [y()], [y()], copies=[x]), "twice"),
            (lambda: step([x[:300], x[299:]], [y()[:300], y()[:213]], [y()[:300], y()[:213]], [y()[:300], y()[:213]]), "twice"),
            (lambda: step([x.reshape(16, 32).t()], [y()], [y()], [y()]), "contiguous"),
            (lambda: step([x], [torch.zeros(1024, device="cuda")[::2]], [y()], [y()]), "contiguous"),
            (lambda: step([x], [y()[:511]], [y()], [y()]), "elements"),
            (lambda: step([x.double()], [y()], [y()], [y()]), "must not be"),
            (lambda: step([x], [y()], [y().bfloat16()], [y()]), "must not be"),
            (lambda: step([x], [y()], [f8()], [f8()]), "must not be"),
            (lambda: step([x], [y()], [y()], [y()], scales=([e8()], [e8()])), "must not be"),
            (lambda: step([x], [y()], [f8()], [f8()], scales=([e8(1)], [e8()])), "elements"),
            (lambda: step([x], [y()], [y()], [y()], clamped=[y().half()]), "must not be"),
            (lambda: step([x], [y()], [y()], [y()], bounds=(1, -1)), "bounds"),
            (lambda: uf.adamw_step([x], [y()], [y()], [y()], torch.zeros(1, device="cuda"), LR), "must not be"),
            (lambda: uf.adamw_step([x, y().half()], [y(), y()], [y(), y()], [y(), y()], torch.zeros(1, device="cuda", dtype=torch.int64), LR), "same types"),
            (lambda: step([x], [y().cpu()], [y()], [y()]), "GPU")):
        with pytest.raises(RuntimeError, match=words):
            call()
    assert (x == 0).all()
    with pytest.raises(TypeError):
        step([x], [None], [y()], [y()])


def test_versions(uf):
    """who watches a tensor sees the write"""
    x, g, m, v, c, d = (torch.ones(10, device="cuda") for _ in range(6))
    before = [t._version for t in (x, g, m, v, c, d)]
    uf.adamw_step([x], [g], [m], [v], 1, LR, copies=[c], clamped=[d])
    assert [t._version - b for t, b in zip((x, g, m, v, c, d), before)] == [1, 0, 1, 1, 1, 1]


# ---------------------------------------------------------------- the optimiser

def small_model(seed=0, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(33, 70), torch.nn.ReLU(), torch.nn.Linear(70, 5)).cuda().to(dtype)


def run_steps(model, optimizer, steps, seed=1):
    g = torch.Generator().manual_seed(seed)
    for _ in range(steps):
        x = torch.randn(16, 33, generator=g).cuda().to(next(model.parameters()).dtype)
        optimizer.zero_grad()
        model(x).square().mean().backward()
        optimizer.step()


def test_optimiser_agrees_with_pytorchs(uf):
    from geo_amd import network
    ours, theirs = small_model(), small_model()
    run_steps(ours, network.AdamW(ours.parameters(), lr=1e-2, weight_decay=0.1), 5)
    run_steps(theirs, torch.optim.AdamW(theirs.parameters(), lr=1e-2, weight_decay=0.1), 5)
    for a, b in zip(ours.parameters(), theirs.parameters()):
        # both round at every step; where a gradient is near 1e-8 its sign and size are rounding's: 5 lr at most
        assert (a - b).abs().max() <= 5e-2 and (a - b).abs().mean() <= 5 * 32 * U


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_optimiser_state_goes_through_a_dict(uf, bits, capturable):
    from geo_amd import network
    for dtype in (torch.float32, torch.bfloat16):
        a, b = small_model(0, dtype), small_model(5, dtype)
        make = lambda m: network.AdamW(m.parameters(), lr=1e-2, state_bits=bits, capturable=capturable)   # noqa: E731
        first, second = make(a), make(b)
        run_steps(a, first, 3)
        b.load_state_dict(a.state_dict())
        second.load_state_dict(first.state_dict())
        run_steps(a, first, 3, seed=2)
        run_steps(b, second, 3, seed=2)
        assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))
        # options come from the dict, as PyTorch's optimisers have it, the kind of the states among them
        third = network.AdamW(a.parameters(), state_bits=40 - bits)
        third.load_state_dict(first.state_dict())
        assert third.param_groups[0]["state_bits"] == bits
        broken = first.state_dict()
        broken["state"][0]["exp_avg"] = broken["state"][0]["exp_avg"].reshape(-1)[1:]
        with pytest.raises(ValueError, match="does not fit"):
            third.load_state_dict(broken)


def test_parameters_without_gradients_and_late_ones(uf):
    from geo_amd import network
    p = [torch.ones(10, device="cuda", requires_grad=True) for _ in range(3)]
    opt = network.AdamW(p, lr=0.1, weight_decay=0.0)
    p[0].grad = torch.ones(10, device="cuda")
    opt.step()
    p[1].grad = torch.ones(10, device="cuda")
    opt.step()
    # the first has made two steps, the second one, the third none; every step of a constant gradient is lr
    for t, want in zip(p, (0.8, 0.9, 1.0)):
        assert (t - want).abs().max() <= 1e-6
    assert not opt.state[p[2]]


def test_training_step_of_the_sc_network(uf):
    """masters, scaled gradients, copies and weight_org in the optimiser's kernel: the same bits as one operation after the other"""
    from geo_amd import network
    torch.manual_seed(3)
    x, y = torch.rand(8, 3, 32, 32).cuda(), torch.randint(10, (8,)).cuda()
    results = []
    for fused in (True, False):
        torch.manual_seed(4)
        net = network.CONV_tiny_add_partial().cuda()
        net.fused_blocks = True
        masters = network.make_param_copies(net)
        opt = network.AdamW(masters, lr=1e-2, weight_decay=0.05)
        stepper = opt if fused else type("Plain", (), {"step": lambda self: opt.step(), "zero_grad": lambda self: opt.zero_grad()})()
        losses = [network.train_step(net, x.clone(), y, torch.nn.CrossEntropyLoss(), stepper, masters) for _ in range(3)]
        results.append([t.clone() for t in losses + masters + list(net.parameters()) + list(net.buffers())])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_training_step(uf, bits):
    from geo_amd import network
    torch.manual_seed(3)
    x, y = torch.rand(8, 3, 32, 32).cuda(), torch.randint(10, (8,)).cuda()
    results = []
    for recorded in (True, False):
        torch.manual_seed(4)
        net = network.CONV_tiny_add_partial().cuda()
        net.fused_blocks = True
        masters, criterion = network.make_param_copies(net), torch.nn.CrossEntropyLoss()
        opt = network.AdamW(masters, lr=1e-2, capturable=True, state_bits=bits)
        step = network.GraphedTrainStep(net, criterion, opt, masters, x, y) if recorded else \
            (lambda a, b: network.train_step(net, a.clone(), b, criterion, opt, masters))
        losses = [step(x, y).clone() for _ in range(4)]
        results.append([t.clone() for t in losses + masters + list(net.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_command_line(uf, tmp_path):
    from geo_amd import main_conv
    for name in ("AdamW", "AdamW8"):
        got = main_conv.main(["--dataset", "SYNTHETIC", "--err", "5555", "--epochs", "1", "--iterations", "2", "--synthetic_size", "256", "--optim", name,
                              "--save_dir", str(tmp_path / name), "--load_unit", "2222", "--load_wait", "2222"])
        assert math.isfinite(got["history"][0]["train_loss"])


def test_step_on_the_host_is_not_recorded(uf):
    """its number would be in the graph, the same in every replay"""
    from geo_amd import network
    p = torch.ones(10, device="cuda", requires_grad=True)
    p.grad = torch.ones(10, device="cuda")
    opt = network.AdamW([p])
    opt.step()
    with pytest.raises(RuntimeError, match="capturable"):
        graph_of(opt.step)
    torch.cuda.synchronize()
    assert opt.state[p]["step"] == 1


def test_first_step_is_not_recorded(uf):
    """it makes the states, which every replay would clear"""
    from geo_amd import network
    p = torch.ones(10, device="cuda", requires_grad=True)
    p.grad = torch.ones(10, device="cuda")
    opt = network.AdamW([p], capturable=True)
    with pytest.raises(RuntimeError, match="first step"):
        graph_of(opt.step)
    torch.cuda.synchronize()
    opt.step()
    graph = graph_of(opt.step)   # (records a step, does not make it)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert opt.state[p]["step"].item() == 4


def test_refused_step_is_not_counted(uf):
    from geo_amd import network
    p = torch.ones(10, device="cuda", requires_grad=True)
    p.grad = torch.ones(10, device="cuda")
    opt = network.AdamW([p])
    opt.step()
    with pytest.raises(RuntimeError, match="copies"):
        opt.step(copies={p: torch.ones(9, device="cuda")})
    assert opt.state[p]["step"] == 1


def test_gradients_that_would_be_written_over(uf):
    memory = torch.ones(64, device="cuda")
    m, v = torch.zeros(16, device="cuda"), torch.zeros(16, device="cuda")
    for begin in (0, 8, 15):
        with pytest.raises(RuntimeError, match="none of its gradients"):
            uf.adamw_step([memory[15:31]], [memory[begin:begin + 16]], [m], [v], 1, 0.1)
    for begin in (31, 32, 48):   # beside the parameter, and one gradient for two
        uf.adamw_step([memory[15:31]], [memory[begin:begin + 16]], [m], [v], 1, 0.1)
    other = [torch.zeros(16, device="cuda") for _ in range(5)]
    uf.adamw_step([memory[15:31], other[0]], [memory[32:48]] * 2, [m, other[1]], [v, other[2]], 1, 0.1)


def test_inference_tensors(uf):
    with torch.inference_mode():
        x, m, v = (torch.zeros(10, device="cuda") for _ in range(3))
        uf.adamw_step([x], [torch.ones(10, device="cuda")], [m], [v], 1, 0.1, weight_decay=0.0)
    assert (x + 0.1).abs().max() < 1e-6
    with pytest.raises(RuntimeError, match="inference"):
        uf.adamw_step([x], [torch.ones(10, device="cuda")], [m], [v], 2, 0.1)
    assert (x + 0.1).abs().max() < 1e-6   # nothing written


def test_masters_that_the_optimiser_does_not_have_are_copied_back(uf):
    from geo_amd import network
    model = small_model()
    masters = network.make_param_copies(model)
    opt = network.AdamW(masters[:2], lr=0.1, weight_decay=0.0)
    for p in model.parameters():
        p.grad = torch.full_like(p, 128.0)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(5.0)   # as a layer's quantisation: the step brings the masters' values back
    network.apply_update(model, opt, masters)
    for i, (master, p) in enumerate(zip(masters, model.parameters())):
        assert torch.equal(master, p) and (master.grad is None)
    assert sum(bool(opt.state[m]) for m in masters[:2]) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_through_a_file(uf, bits, tmp_path):
    from geo_amd import network
    a, b = small_model(0), small_model(0)
    first, second = network.AdamW(a.parameters(), state_bits=bits), network.AdamW(b.parameters(), state_bits=bits)
    run_steps(a, first, 2)
    b.load_state_dict(a.state_dict())
    torch.save(first.state_dict(), tmp_path / "state.pt")
    second.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    run_steps(a, first, 2, seed=3)
    run_steps(b, second, 2, seed=3)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))


def test_several_groups_and_types(uf):
    """groups of their own rates and states; parameters of several types in one"""
    from geo_amd import network
    p = [torch.ones(300, device="cuda", dtype=t, requires_grad=True) for t in (torch.float32, torch.bfloat16, torch.float16, torch.float32)]
    opt = network.AdamW([dict(params=p[:3], lr=0.5), dict(params=p[3:], lr=0.25, state_bits=8)], weight_decay=0.0)
    for t in p:
        t.grad = torch.full_like(t, 0.5)
    opt.step()
    for t, want in zip(p, (0.5, 0.5, 0.5, 0.75)):
        assert (t.float() - want).abs().max() <= 2 ** -8
    assert opt.state[p[3]]["exp_avg"].dtype == torch.float8_e4m3fn and opt.state[p[1]]["exp_avg"].dtype == torch.float32
