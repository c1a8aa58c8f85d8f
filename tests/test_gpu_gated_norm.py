"""The norm behind a block, its gate, the scaled residual and the next norm, against their formulas in 64 bits.

Tolerances follow from the roundings: U = 2^-24 is half a unit of fp32, EPS the half unit of an output's type.  A row's sum of squares
goes through at most cols / 64 + 64 additions, a mean of products too; a handful of products round once each.  With K U for all that
one stage does, and `spread` for how much larger the parts of a total are than the total itself, each stage's error is at most
K U (1 + spread) of the sum of its terms' magnitudes; four stages follow each other in the backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half of a type's smallest step
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def uf():
    assert torch.cuda.is_available(), "these tests need the GPU"
    from geo_amd import utils_functional as m
    return m


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def close(got, want, tolerance):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bad = ((got - want).abs() > tolerance) & ~torch.isnan(want)
    assert not bad.any(), (int(bad.sum()), ((got - want).abs() / tolerance)[bad].max().item())


def inputs(rows, cols, dtype, runs=None, post=True, scale=True, seed=0, shape=None):
    """x, residual, weight, post, gate, scale; runs: None no gate, 1 a gate per channel, else one per run of rows"""
    around = lambda k, *s: (1 + rand(*s, seed=seed + k, scale=0.2)).to(dtype)   # noqa: E731
    x = rand(rows, cols, dtype=dtype, seed=seed + 1, scale=2.0)
    residual = rand(rows, cols, dtype=dtype, seed=seed + 2)
    gate = None if runs is None else rand(cols, dtype=dtype, seed=seed + 3) if runs == 1 else rand(runs, cols, dtype=dtype, seed=seed + 3)
    return dict(x=x, residual=residual, weight=around(4, cols), post=around(5, cols) if post else None, gate=gate,
                scale=around(6, cols) if scale else None)


def call(uf, v, eps, eight=None):
    x, residual, gate = v["x"], v["residual"], v["gate"]
    if gate is not None and gate.dim() == 2:
        x, residual, gate = (t.unflatten(0, (gate.shape[0], -1)) for t in (x, residual, gate))   # gate: (runs, 1, columns)
    rest = dict(post_weight=v["post"], gate=gate, residual_scale=v["scale"], eps=eps)
    got = uf.gated_norm(x, residual, v["weight"], **rest) if eight is None else uf.gated_norm_q8(x, residual, v["weight"], values=eight, **rest)
    return [t.flatten(0, 1) if t is not None and t.dim() == 3 else t for t in got]


def formulas(v, eps, g=None, h=None):
    """outputs and gradients written out in 64 bits, each with its tolerance"""
    w = {k: t.double() if t is not None else None for k, t in v.items()}
    dtype, (rows, cols) = v["x"].dtype, v["x"].shape
    half, tiny, k = EPS[dtype], TINY[dtype], (cols / 64 + 64 + 16) * U
    ones = torch.ones(cols, dtype=torch.float64, device="cuda")
    post, scale = (w[n] if w[n] is not None else ones for n in ("post", "scale"))
    gate = w["gate"].reshape(-1, cols) if w["gate"] is not None else ones[None]
    gate = gate.repeat_interleave(rows // gate.shape[0], 0)
    mean = lambda t: t.mean(-1, keepdim=True)   # noqa: E731
    r1 = (mean(w["x"].square()) + eps).rsqrt() if w["post"] is not None else torch.ones(rows, 1, dtype=torch.float64, device="cuda")
    n1 = w["x"] * r1
    m = n1 * post
    total = scale * w["residual"] + gate * m
    parts = (scale * w["residual"]).abs() + (gate * m).abs()
    r2 = (mean(total.square()) + eps).rsqrt()
    n2, n2_parts = total * r2, parts * r2
    spread = (mean(parts.square()) / mean(total.square()).clamp(min=1e-300)).sqrt().clamp(max=1e6)
    k = k * (1 + spread)
    out = {"total": (total, half * total.abs() + k * parts + tiny),
           "out": (n2 * w["weight"], half * (n2 * w["weight"]).abs() + 2 * k * (n2_parts + n2.abs()) * w["weight"].abs() + tiny)}
    if g is None:
        return out
    g, h = g.double(), h.double() if h is not None else torch.zeros_like(g)
    u = g * w["weight"]
    dt = r2 * (u - n2 * mean(u * n2)) + h
    dt_parts = r2 * (u.abs() + n2_parts * mean(u.abs() * n2_parts)) + h.abs()
    e, e_parts = dt * gate, dt_parts * gate.abs()
    s, s_parts = e * post, e_parts * post.abs()
    has_post = w["post"] is not None
    dx = r1 * (s - n1 * mean(s * n1)) if has_post else s
    dx_parts = r1 * (s_parts + n1.abs() * mean(s_parts * n1.abs())) if has_post else s_parts
    runs = (lambda t: t.reshape(-1, rows, cols).sum(1)[0] if v["gate"].dim() == 1 else t.reshape(v["gate"].shape[0], -1, cols).sum(1))
    down = rows * U   # additions of a sum over rows
    grads = {"x": (dx, dx_parts), "residual": (dt * scale, dt_parts * scale.abs())}
    sums = {"weight": (g * n2, g.abs() * n2_parts)}
    if has_post:
        sums["post"] = (e * n1, e_parts * n1.abs())
    if w["scale"] is not None:
        sums["scale"] = (dt * w["residual"], dt_parts * w["residual"].abs())
    for name, (value, size) in grads.items():
        out["d" + name] = (value, half * value.abs() + 4 * k * size + tiny)
    for name, (value, size) in sums.items():
        value, size = value.sum(0), ((4 * k + down) * size).sum(0)
        out["d" + name] = (value, half * value.abs() + size + tiny)
    if w["gate"] is not None:
        value, size = runs(dt * m), runs((4 * k + down) * dt_parts * m.abs())
        out["dgate"] = (value, half * value.abs() + size + tiny)
    return out


def leaves(v):
    return {k: t.clone().requires_grad_(True) if t is not None else None for k, t in v.items()}


def check(uf, v, eps=1e-5, g=None, h=None, want_h=True):
    rows, cols = v["x"].shape
    dtype = v["x"].dtype
    g = rand(rows, cols, dtype=dtype, seed=77) if g is None else g
    h = (rand(rows, cols, dtype=dtype, seed=78) if h is None else h) if want_h else None
    v = leaves(v)
    out, total = call(uf, v, eps)
    names = [k for k, t in v.items() if t is not None]
    outputs, given = ((out, total), (g, h)) if want_h else ((out,), (g,))
    grads = torch.autograd.grad(outputs, [v[k] for k in names], given)
    want = formulas({k: t.detach() if t is not None else None for k, t in v.items()}, eps, g, h)
    got = dict(out=out.detach(), total=total.detach(), **{"d" + k: t for k, t in zip(names, grads)})
    for name, t in got.items():
        assert t.dtype == dtype
        close(t, *want[name])
    with torch.no_grad():   # without a graph, the same bits
        for a, b in zip(call(uf, v, eps), (out, total)):
            assert torch.equal(a, b)
    return got


# one element, parts of a chunk, half a wave, a wave, several; the limits of what a workgroup holds in either direction, and beyond
SHAPES = [(1, 1), (3, 7), (5, 8), (70, 256), (9, 257), (2, 511), (600, 513), (1, 4096), (4, 8191), (2, 8192), (3, 8200), (2, 32768), (2, 40007)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(uf, dtype, shape):
    check(uf, inputs(*shape, dtype, runs=1))
    check(uf, inputs(*shape, dtype, runs=shape[0] if shape[0] > 1 else None))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("runs", [None, 1, 3])
@pytest.mark.parametrize("shape", [(33, 100), (33, 1000), (33, 9000)])
def test_parts_that_are_not_there(uf, post, scale, runs, shape):
    for dtype in (torch.float32, torch.bfloat16):
        check(uf, inputs(*shape, dtype, runs=runs, post=post, scale=scale))
    check(uf, inputs(*shape, torch.float32, runs=runs, post=post, scale=scale), want_h=False)


# rows, columns and runs: several runs in a unit's rows, runs cut once and many times, in the middle of a unit and at its border
@pytest.mark.parametrize("case", [(5000, 600, 50), (5000, 600, 2500), (5000, 600, 1000), (5000, 600, 625), (5000, 600, 5000), (5000, 600, 2),
                                  (2100, 40, 700), (6300, 40, 900), (6300, 300, 3), (300, 8200, 100), (300, 8200, 60), (300, 8200, 2), (513, 600, 171)])
def test_runs_of_rows_that_share_a_gate(uf, case):
    rows, cols, runs = case
    for dtype in (torch.float32, torch.float16):
        check(uf, inputs(rows, cols, dtype, runs=runs, seed=runs))


@pytest.mark.parametrize("eight", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_eight_bits(uf, eight, shape):
    """the next norm's rows in 8 bits: within half a step and what n itself may be off"""
    for dtype in TYPES:
        v = inputs(*shape, dtype, runs=1)
        with torch.no_grad():
            q, scale, total, values = call(uf, v, 1e-5, eight)
            assert torch.equal(total, call(uf, v, 1e-5)[1])
        n, off = formulas({k: t.float() if t is not None else None for k, t in v.items()}, 1e-5)["out"]
        a = n.abs().amax(-1)
        slack = (off / a[:, None].clamp(min=1e-30)).amax(-1)
        assert ((scale.double() - a / 127).abs() <= (slack + 4 * U) * a / 127).all()
        steps = n * torch.where(a > 0, 127 / a, 0.0)[:, None]
        assert ((q.double() - steps).abs() <= 0.5 + 127 * (4 * U + 2 * slack[:, None])).all()
        want = q.double() * scale.double()[:, None]
        close(values, want, (EPS[eight] + U) * want.abs() + TINY[eight])
    # the products take it as it is
    w = rand(24, shape[1], seed=9)
    wq, ws, _ = uf.quantize_rows(w)
    y = uf.matmul_q8(q, scale, wq, ws)
    exact = (q.double() @ wq.double().t()) * scale.double()[:, None] * ws.double()
    close(y, exact, 4 * U * exact.abs() + 1e-300)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(uf, dtype):
    """rows of other distances, at odd addresses; expanded gradients"""
    rows, cols = 21, 515
    base = inputs(rows, cols, dtype, runs=1)
    want = check(uf, base)
    wide = {k: torch.full((rows, cols + 7), 9.0, dtype=dtype, device="cuda") for k in ("x", "residual", "g", "h")}
    other = {}
    for k in wide:
        other[k] = wide[k][:, 3:3 + cols]
    other["x"].copy_(base["x"])
    other["residual"].copy_(base["residual"])
    other["g"].copy_(rand(rows, cols, dtype=dtype, seed=77))
    other["h"].copy_(rand(rows, cols, dtype=dtype, seed=78))
    v = dict(base, x=other["x"].detach().requires_grad_(True), residual=other["residual"].detach().requires_grad_(True))
    packed = torch.zeros(4, cols + 1, dtype=dtype, device="cuda")
    for i, k in enumerate(("weight", "post", "gate", "scale")):
        packed[i, 1:].copy_(base[k])
        v[k] = packed[i, 1:].detach().requires_grad_(True)
    out, total = uf.gated_norm(v["x"], v["residual"], v["weight"], v["post"], v["gate"], v["scale"], 1e-5)
    assert torch.equal(out, want["out"]) and torch.equal(total, want["total"])
    grads = torch.autograd.grad((out, total), [v[k] for k in ("x", "residual", "weight", "post", "gate", "scale")], (other["g"], other["h"]))
    for k, t in zip(("x", "residual", "weight", "post", "gate", "scale"), grads):
        assert torch.equal(t, want["d" + k]), k
    assert all((wide[k][:, :3] == 9).all() and (wide[k][:, 3 + cols:] == 9).all() for k in wide)
    # one gradient for all rows, and for all elements
    one = rand(1, cols, dtype=dtype, seed=5).expand(rows, cols)
    check(uf, base, g=one, h=torch.ones(1, 1, dtype=dtype, device="cuda").expand(rows, cols))
    # other orders and dimensions
    x = base["x"].t().contiguous().t()
    assert torch.equal(uf.gated_norm(x, base["residual"], base["weight"])[0], uf.gated_norm(base["x"], base["residual"], base["weight"])[0])
    a, b = uf.gated_norm(base["x"].reshape(3, 7, cols), base["residual"].reshape(3, 7, cols), base["weight"])
    assert a.shape == b.shape == (3, 7, cols)


def test_gates_of_any_leading_dimensions(uf):
    x, residual, w = rand(4, 3, 5, 40, seed=1), rand(4, 3, 5, 40, seed=2), rand(40, seed=3)
    for shape in ((40,), (1, 1, 1, 40), (4, 1, 1, 40), (4, 3, 1, 40), (4, 3, 5, 40)):
        gate = rand(*shape, seed=4).requires_grad_(True)
        out, total = uf.gated_norm(x, residual, w, gate=gate)
        assert torch.allclose(total, residual + gate * x, rtol=1e-6, atol=1e-6)
        d, = torch.autograd.grad((total,), (gate,), (residual,))
        want = (residual.double() * x.double()).reshape(-1, 40)
        want = want.reshape(-1, 60 // max(1, gate.numel() // 40), 40).sum(1).reshape(shape)
        assert d.shape == gate.shape
        close(d, want, 80 * U * (residual * x).abs().double().sum())
    for shape in ((1, 3, 1, 40), (4, 1, 5, 40), (3, 1, 1, 40), (4, 1, 40), (4, 3, 5, 1), (39,)):
        with pytest.raises(RuntimeError, match="gate must"):
            uf.gated_norm(x, residual, w, gate=rand(*shape))


def test_rows_of_any_magnitude(uf):
    """squares beyond fp32's range on either side, in either norm"""
    cols = 300
    for size in (1e25, 1e-25):
        for width in (cols, 9000, 40000):
            v = inputs(6, width, torch.float32, runs=1)
            v["x"] = v["x"] * torch.tensor([1.0, size, 1.0, size, 1.0, size], device="cuda")[:, None]
            v["residual"] = v["residual"] * torch.tensor([1.0, size, size, 1.0, 1.0, size], device="cuda")[:, None]
            if size < 1:   # (the gated branch would hide the residual)
                v["post"] = None
            g = torch.ones(6, width, device="cuda") * 1e-3
            check(uf, v, eps=0.0, g=g, h=g)
            q, scale, _, values = call(uf, {k: t.detach() if t is not None else None for k, t in v.items()}, 0.0, torch.float32)
            n = formulas(v, 0.0)["out"][0]
            assert ((values.double() - n).abs() <= n.abs().amax(-1, keepdim=True) / 127 * 0.51).all()


def test_rows_that_hold_no_numbers(uf):
    """stay by themselves"""
    for dtype in TYPES:
        for shape in ((7, 300), (7, 9000), (7, 40000)):
            v = inputs(*shape, dtype, runs=1)
            good = call(uf, v, 1e-6), call(uf, v, 1e-6, torch.float32)
            for row, k, value in ((1, "x", float("nan")), (3, "residual", float("inf")), (4, "x", -float("inf"))):
                v[k][row, 5] = value
            v["x"][6], v["residual"][6] = 0.0, 0.0
            out, total = call(uf, v, 1e-6)
            q, scale, total8, values = call(uf, v, 1e-6, torch.float32)
            for row in (0, 2, 5):
                assert torch.equal(out[row], good[0][0][row]) and torch.equal(values[row], good[1][3][row])
            assert torch.isnan(out[1]).all() and torch.isnan(out[3, 5]) and torch.isnan(out[4, 5])
            assert torch.isnan(scale[[1, 3, 4]]).all() and (q[[1, 3, 4]] == 0).all()
            assert (out[6] == 0).all() and (total[6] == 0).all() and (values[6] == 0).all() and scale[6] == 0


def test_some_gradients_only(uf):
    v = inputs(50, 300, torch.float32, runs=5)
    g = rand(50, 300, seed=3)
    every = check(uf, v, g=g, want_h=False)
    for name in ("x", "residual", "weight", "post", "gate", "scale"):
        one = {k: t.clone().requires_grad_(k == name) for k, t in v.items()}
        d, = torch.autograd.grad((call(uf, one, 1e-5)[0],), (one[name],), (g,))
        assert torch.equal(d, every["d" + name])
    # of the sum alone; of nothing that the loss depends on
    one = leaves(v)
    total = call(uf, one, 1e-5)[1]
    d = torch.autograd.grad(total, [one["residual"], one["weight"]], g, allow_unused=True)
    assert torch.equal(d[0], (g * v["scale"])) and (d[1] == 0).all()


def test_gradients_against_differences(uf):
    v = {k: t.double().float() if t is not None else None for k, t in inputs(6, 40, torch.float32, runs=2).items()}
    g, h = rand(6, 40, seed=1).double(), rand(6, 40, seed=2).double()
    got = check(uf, v, g=g.float(), h=h.float())

    for name in ("x", "residual", "weight", "post", "gate", "scale"):
        wide = {k: t.double() for k, t in v.items()}
        direction = rand(*v[name].shape, seed=8).double()
        step = 1e-5
        ends = []
        for sign in (1, -1):
            moved = dict(wide)
            moved[name] = wide[name] + sign * step * direction
            ends.append(loss_in_64(moved, g, h))
        want = ((ends[0] - ends[1]) / (2 * step)).item()
        have = (got["d" + name].double() * direction).sum().item()
        # fp32 gradients: some 100 U of the sum of magnitudes; the difference: its third derivative's step^2
        assert abs(have - want) <= 200 * U * (got["d" + name].double() * direction).abs().sum().item() * 10 + 1e-6 * abs(want)


def loss_in_64(v, g, h):
    rows, cols = v["x"].shape
    gate = v["gate"].repeat_interleave(rows // v["gate"].shape[0], 0)
    unit = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()   # noqa: E731
    total = v["scale"] * v["residual"] + gate * (unit(v["x"]) * v["post"])
    return (unit(total) * v["weight"] * g + total * h).sum()


def test_no_rows(uf):
    x, w = torch.zeros(0, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda", requires_grad=True)
    out, total = uf.gated_norm(x, x, w, post_weight=w, gate=w, residual_scale=w)
    assert out.shape == total.shape == (0, 40)
    d = torch.autograd.grad((out.sum() + total.sum(),), (x, w))
    assert d[0].shape == x.shape and (d[1] == 0).all()
    with torch.no_grad():
        q, scale, _, values = uf.gated_norm_q8(x, x, w, values=torch.float32)
    assert q.shape == (0, 40) and scale.shape == (0,)


def test_same_bits_on_every_run(uf):
    v = inputs(3000, 1000, torch.bfloat16, runs=30)
    first = check(uf, v)
    for _ in range(3):
        again = check(uf, v)
        assert all(torch.equal(first[k], again[k]) for k in first)


def test_replayed_and_on_another_stream(uf):
    v = leaves(inputs(100, 700, torch.float32, runs=4))
    names = ("x", "residual", "weight", "post", "gate", "scale")
    g = rand(100, 700, seed=4)

    def step():
        out, total = call(uf, v, 1e-5)
        return [out, total] + list(torch.autograd.grad((out, total), [v[k] for k in names], (g, g)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.detach().clone() for t in step()]   # (no graph of these leaves lives while one is recorded)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        with torch.no_grad():
            v["x"].mul_(1.25)
            v["gate"].add_(0.1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_refusals(uf):
    x, w = torch.zeros(4, 40, device="cuda"), torch.ones(40, device="cuda")
    for bad, words in ((dict(residual=x[:3]), "shape and type"), (dict(residual=x.half()), "shape and type"), (dict(weight=w[:39]), "40 elements"),
                       (dict(weight=w.half()), "type of x"), (dict(post_weight=w[None]), "40 elements"), (dict(residual_scale=w.double()), "type of x"),
                       (dict(gate=w.half()), "type of x"), (dict(eps=-1.0), "eps"), (dict(x=x.double()), "float32"), (dict(x=x.cpu()), "GPU"),
                       (dict(gate=w.cpu()), "GPU"), (dict(x=x[:, :0]), "no elements")):
        args = dict(dict(x=x, residual=x, weight=w), **bad)
        with pytest.raises(RuntimeError, match=words):
            uf.gated_norm(**args)
        with pytest.raises(RuntimeError, match=words):
            uf.gated_norm_q8(**args)
    y = x.clone().requires_grad_(True)
    with pytest.raises(ValueError, match="no gradients"):
        uf.gated_norm_q8(y, x, w)
    out, total = uf.gated_norm(y, x, w)
    d, = torch.autograd.grad(out.sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(d.sum(), y)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: uf.gated_norm(t, t, w)[0], (x,))
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            uf.gated_norm(fw.make_dual(x, x), x, w)
