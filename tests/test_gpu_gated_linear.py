"""A layer behind a gated norm: what it gives in training and from a prepared weight is the same bits in every type, because the norm goes
from fp32 to 8 bits in both; its gradients are the norm's and the product's."""
import pytest
import torch

from tests.test_gpu_dense import EPS, TYPES, U, close, product64, subnormal, uf  # noqa: F401
from tests.test_gpu_dense_epilogue import act64
from tests.test_gpu_gated_norm import call, inputs, leaves, rand

pytestmark = pytest.mark.gpu


# two rows in a wave, one, several waves, two rows at once, rows that are read again
@pytest.mark.parametrize("shape", [(1, 8, 5), (9, 48, 20), (130, 600, 70), (2051, 1100, 33), (3, 32776, 17)])
@pytest.mark.parametrize("dtype", TYPES)
def test_training_and_serving_agree(uf, dtype, shape):
    from geo_amd import utils_class
    rows, cols, out = shape
    torch.manual_seed(rows)
    layer = utils_class.GatedNormLinear_Q8(cols, out, bias=True, activation="gelu").cuda()
    with torch.no_grad():
        for p in layer.parameters():
            p.add_(torch.randn_like(p) * 0.2)
    layer.to(dtype)
    x, residual = rand(rows, cols, dtype=dtype, seed=1), rand(rows, cols, dtype=dtype, seed=2)
    y, total = layer(x, residual)
    assert y.requires_grad and total.requires_grad
    with torch.no_grad():
        plain = layer(x, residual)
        layer.prepare()
        served = layer(x, residual)
    for got in (plain, served):
        assert torch.equal(got[0], y) and torch.equal(got[1], total)
    assert torch.equal(layer(x, residual)[0], y)   # (a call with gradients rounds anew)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(6, 40, 24, 1), (12, 300, 30, 4), (70, 513, 64, None), (2050, 1100, 20, 5), (4, 9000, 12, 2)])
def test_gradients(uf, dtype, case):
    """without an activation the gradient of the norm's output does not depend on the rows: the same bits as the norm by itself has from it"""
    rows, cols, n, runs = case
    v = leaves(inputs(rows, cols, dtype, runs=runs))
    w = rand(n, cols, dtype=dtype, seed=11, scale=cols ** -0.5).requires_grad_(True)
    bias = rand(n, dtype=dtype, seed=12).requires_grad_(True)
    g, h = rand(rows, n, dtype=dtype, seed=13), rand(rows, cols, dtype=dtype, seed=14)
    shape = (lambda t: t.unflatten(0, (runs, -1))) if runs and runs > 1 else (lambda t: t)
    gate = shape(v["gate"]) if runs and runs > 1 else v["gate"]
    y, total = uf.gated_norm_linear_q8(shape(v["x"]), shape(v["residual"]), v["weight"], w, post_weight=v["post"], gate=gate,
                                       residual_scale=v["scale"], eps=1e-5, bias=bias)
    y, total = (t.reshape(rows, -1) for t in (y, total))
    names = [k for k, t in v.items() if t is not None]
    got = torch.autograd.grad((y, total), [v[k] for k in names] + [w, bias], (g, h))
    with torch.no_grad():
        q, s, same, _ = call(uf, v, 1e-5, torch.float32)
        s = s.reshape(-1)
        wq, ws, _ = uf.quantize_rows(w)
        assert torch.equal(total, same)
        assert torch.equal(y, uf.matmul_q8(q, s, wq, ws, dtype=dtype, bias=bias))
    some = rand(rows, cols, dtype=dtype, seed=15).requires_grad_(True)
    dn, = torch.autograd.grad(uf.linear_q8(some, w.detach()), some, g)
    want = torch.autograd.grad(call(uf, v, 1e-5), [v[k] for k in names], (dn, h))
    for name, a, b in zip(names, got, want):
        assert torch.equal(a, b), name
    # the weight's: (g scale)^T q, each of the scaled gradient's terms an fp16 number
    xr, g64 = q.double() * s.double()[:, None], g.double()
    kept = EPS[torch.float16] ** (1 if dtype == torch.bfloat16 else 2) + U
    size, dw = g64.abs().t() @ xr.abs(), g64.t() @ xr
    low = 2.0 ** -39 * (g64 * s.double()[:, None]).abs().amax(0)[:, None] * q.double().abs().sum(0)
    close(got[-2], dw, EPS[dtype] * dw.abs() + (kept + 4 * rows * U) * size + low + subnormal(dtype))
    close(got[-1], g64.sum(0), EPS[dtype] * g64.sum(0).abs() + rows * U * g64.abs().sum(0) + subnormal(dtype))


@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
def test_gradients_with_an_activation(uf, kind):
    """dz = g slope is off by some 20 U of itself; the products by that and their own sums (as the norm's own layer is held to)"""
    v, w, bias = leaves(inputs(100, 96, torch.float32, runs=4)), rand(72, 96, seed=3, scale=0.1).requires_grad_(True), rand(72, seed=4).requires_grad_(True)
    g, h = rand(100, 72, seed=6), rand(100, 96, seed=7)
    around = dict(post_weight=v["post"], gate=v["gate"].unsqueeze(1), residual_scale=v["scale"], eps=1e-5)
    names = list(v)
    three = lambda t: t.unflatten(0, (4, 25))   # noqa: E731
    one = uf.gated_norm_linear_q8(three(v["x"]), three(v["residual"]), v["weight"], w, bias=bias, activation=kind, **around)
    got = torch.autograd.grad(one, [v[k] for k in names] + [w, bias], (three(g), three(h)))
    with torch.no_grad():
        q, s, _, _ = call(uf, v, 1e-5, torch.float32)
        s = s.reshape(-1)
        wq, ws, _ = uf.quantize_rows(w)
        slope = act64(product64(q, s, wq, ws) + bias.double(), kind)[1]
    dz = (g.double() * slope).float()
    two = uf.gated_norm_linear_q8(three(v["x"]), three(v["residual"]), v["weight"], w, bias=bias, **around)
    want = torch.autograd.grad(two, [v[k] for k in names] + [w, bias], (three(dz), three(h)))
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_some_gradients_only(uf):
    v, w, bias = inputs(60, 200, torch.float32, runs=3), rand(30, 200, seed=3, scale=0.1), rand(30, seed=4)
    everything = dict(v, w=w, bias=bias)
    g, h = rand(60, 30, seed=5), rand(60, 200, seed=6)

    def run(t):
        shape = lambda a: a.unflatten(0, (3, 20))   # noqa: E731
        y, total = uf.gated_norm_linear_q8(shape(t["x"]), shape(t["residual"]), t["weight"], t["w"], post_weight=t["post"], gate=t["gate"].unsqueeze(1),
                                           residual_scale=t["scale"], bias=t["bias"], activation="silu")
        return y.flatten(0, 1), total.flatten(0, 1)

    of = {k: t.clone().requires_grad_(True) for k, t in everything.items()}
    y, total = run(of)
    all_of = dict(zip(of, torch.autograd.grad((y, total), list(of.values()), (g, h))))
    for name in everything:
        one = {k: t.clone().requires_grad_(k == name) for k, t in everything.items()}
        out = run(one)
        assert out[0].requires_grad
        both = name not in ("w", "bias")   # the sum depends on neither
        d, = torch.autograd.grad(out if both else out[:1], one[name], (g, h) if both else (g,))
        assert torch.equal(d, all_of[name]), name
    # of the sum alone: the layer's are not there
    d = torch.autograd.grad(run(of)[1], list(of.values()), h, allow_unused=True)
    assert all(d[list(of).index(k)] is None for k in ("w", "bias"))
    assert torch.equal(d[list(of).index("residual")], h * v["scale"])


def test_replayed(uf):
    """a pass recorded and replayed, against eager passes on changed inputs"""
    v, w = leaves(inputs(100, 700, torch.float32, runs=1)), rand(50, 700, seed=3, scale=0.1).requires_grad_(True)
    g, h = rand(100, 50, seed=4), rand(100, 700, seed=5)
    held_leaves = [v[k] for k in v] + [w]

    def step():
        out = uf.gated_norm_linear_q8(v["x"], v["residual"], v["weight"], w, post_weight=v["post"], gate=v["gate"], residual_scale=v["scale"], activation="relu")
        return [t.detach() for t in out] + list(torch.autograd.grad(out, held_leaves, (g, h)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        [t.clone() for t in step()]   # (no graph of these leaves lives while one is recorded)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        with torch.no_grad():
            v["x"].mul_(1.25)
            w.add_(0.01)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_refusals_and_no_rows(uf):
    x, gain, w = rand(6, 32, seed=1), rand(32, seed=2), rand(20, 32, seed=3)
    good = dict(x=x, residual=x, gain=gain, weight=w)
    for bad, words in ((dict(residual=x[:5]), "shape and type"), (dict(gain=gain[:31]), "32 elements"), (dict(weight=w[:, :31]), "rows of weight_q 31"),
                       (dict(gate=gain.half()), "type of x"), (dict(activation="tanh"), "activation must"), (dict(bias=gain), "20 elements"),
                       (dict(eps=-1.0), "eps"), (dict(x=x.cpu()), "GPU"), (dict(weight=w.cpu()), "GPU")):
        with pytest.raises(RuntimeError, match=words):
            uf.gated_norm_linear_q8(**dict(good, **bad))
    y = x.clone().requires_grad_(True)
    out, _ = uf.gated_norm_linear_q8(y, x, gain, w)
    d, = torch.autograd.grad(out.sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(d.sum(), y)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            uf.gated_norm_linear_q8(fw.make_dual(x, x), x, gain, w)
    none = torch.zeros(0, 32, device="cuda", requires_grad=True)
    w.requires_grad_(True)
    out, total = uf.gated_norm_linear_q8(none, none, gain, w, activation="gelu")
    assert out.shape == (0, 20) and total.shape == (0, 32)
    d = torch.autograd.grad(out.sum() + total.sum(), (none, w))
    assert d[0].shape == (0, 32) and (d[1] == 0).all()
