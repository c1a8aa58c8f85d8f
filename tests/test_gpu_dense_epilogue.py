"""The 8-bit product with bias, activation and residual in its epilogue, and its gradients, against the formulas in 64 bits.

z: the sum's conversion, two scales and the bias round once each (4 U of the product and the bias).  The activations change by at most 1.13
times what z does, their slopes by at most 0.8 times; erff and expf are allowed four units (8 U) of what they give, the arithmetic
around them as much.  A slope is kept with half a step of fp16 (2^-11, 2^-25 at the least) where x is bf16, else of fp32."""
import math

import pytest
import torch

from tests.test_dense_plan import FEW, SHAPES, STREAMED, TILES
from tests.test_gpu_dense import EPS, PRODUCTS, TYPES, U, close, product64, rand, random_q8, subnormal, uf  # noqa: F401
from tests.test_gpu_dense_kernels import aligned

pytestmark = pytest.mark.gpu

KINDS = [None, "relu", "gelu", "silu"]


def act64(z, kind):
    """the activation and its slope"""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def epilogue64(p, bias, kind, residual, dtype):
    """y, its tolerance; the slope, its tolerance and where z is too near a relu's corner to tell"""
    b = bias.double() if bias is not None else torch.zeros(p.shape[1], dtype=torch.float64, device=p.device)
    z, off = p + b, 4 * U * (p.abs() + b.abs())
    y, d = act64(z, kind)
    r = residual.double() if residual is not None else torch.zeros_like(y)
    tolerance = 1.13 * off + 16 * U * (z.abs() if kind in ("gelu", "silu") else 0 * z) + (EPS[dtype] + U) * (y + r).abs() + U * r.abs() + subnormal(dtype)
    kept, least = (EPS[torch.float16], 2.0 ** -25) if dtype is torch.bfloat16 else (U, 0)
    slope_off = 0.8 * off + 16 * U + kept * d.abs() + least if kind in ("gelu", "silu") else torch.zeros_like(d)
    return y + r, tolerance, d, slope_off, (z.abs() <= off) if kind == "relu" else torch.zeros_like(z, dtype=torch.bool)


def check(uf, q, s, wq, ws, dtype, kind, bias=None, residual=None):
    y = uf.matmul_q8(q, s, wq, ws, dtype=dtype, bias=bias, activation=kind, residual=residual)
    want, tolerance, *_ = epilogue64(product64(q, s, wq, ws), bias, kind, residual, dtype)
    close(y, want, tolerance)


@pytest.mark.parametrize("shape", sorted(set(PRODUCTS) | set(SHAPES)))
def test_kernels(uf, shape):
    """every kernel, tile, cut and edge of the product, with all types and activations among them"""
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 1), random_q8(n, k, 2)
    q, wq, ws = aligned(q), aligned(wq), ws / (k ** 0.5 * 40)   # z of about one
    for i, dtype in enumerate(TYPES):
        kind = KINDS[(m + n + i) % 4]
        bias = rand(n, dtype=TYPES[(i + n) % 3], seed=3) if (n + i) % 3 else None
        residual = rand(m, n, dtype=dtype, seed=4) if (m + i) % 3 or (bias is None and kind is None) else None
        check(uf, q, s, wq, ws, dtype, kind, bias, residual)


# rows and columns just beyond whole tiles, where the tiles are just beyond what all compute units do at once: strips of their own
STRIPS = [(4096, 4099, 300), (4100, 4096, 300), (4111, 4160, 300), (4160, 8192 - 255, 260), (2049, 2051 * 4, 270)]


@pytest.mark.parametrize("shape", STRIPS)
def test_strips(uf, shape):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 1), random_q8(n, k, 2)
    q, wq, ws = aligned(q), aligned(wq), ws / (k ** 0.5 * 40)
    for dtype in TYPES:
        want = product64(q, s, wq, ws)
        close(uf.matmul_q8(q, s, wq, ws, dtype=dtype), want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))
        check(uf, q, s, wq, ws, dtype, "gelu", rand(n, dtype=dtype, seed=3), rand(m, n, dtype=dtype, seed=4))
    # gradients of the same sizes: either product's rows and columns
    g = rand(m, n, dtype=torch.bfloat16, seed=5)
    x, w = rand(m, k, dtype=torch.bfloat16, seed=6), rand(n, k, dtype=torch.bfloat16, seed=7)
    bias = rand(n, seed=8)
    _, (dx, dw, dbias) = gradients(uf, x, w, bias, None, g, "silu")
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    _, _, slope, slope_off, _ = epilogue64(product64(q, s, wq, ws), bias.detach(), "silu", None, torch.bfloat16)
    dz, dz_off = g.double() * slope, g.double().abs() * (slope_off + U * slope.abs())
    xr, wr = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    kept = EPS[torch.float16] + U
    for got, want, size, off, depth in ((dx, dz @ wr, dz.abs() @ wr.abs(), dz_off @ wr.abs(), n),
                                        (dw, dz.t() @ xr, dz.t().abs() @ xr.abs(), dz_off.t() @ xr.abs(), m)):
        close(got, want, EPS[torch.bfloat16] * want.abs() + (kept + 2 * depth * U) * size + off + 1e-9)
    close(dbias, dz.sum(0), U * dz.sum(0).abs() + m * U * dz.abs().sum(0) + dz_off.sum(0))


# columns that end inside a chunk of a tile's first and second half, with fewer than eight of them there, and exactly at their ends
@pytest.mark.parametrize("cols", [1, 7, 8, 9, 31, 32, 33, 39, 40, 41, 63, 64, 65, 100, 127, 128, 129, 200, 257, 263, 264, 385, 391, 392, 500])
@pytest.mark.parametrize("rows,inner", [(66, 260), (129, 70), (1000, 2100)])
def test_columns_that_end_anywhere(uf, rows, cols, inner):
    (q, s), (wq, ws) = random_q8(rows, inner, 1), random_q8(cols, inner, 2)
    q, wq, ws = aligned(q), aligned(wq), ws / (inner ** 0.5 * 40)
    for dtype in TYPES:
        check(uf, q, s, wq, ws, dtype, "gelu", rand(cols, dtype=dtype, seed=3), rand(rows, cols, dtype=dtype, seed=4))


# the same where the tiles are large
@pytest.mark.parametrize("cols", [4100, 4103, 4107, 4200, 4223, 4225, 4230, 4300])
def test_columns_that_end_anywhere_in_large_tiles(uf, cols):
    rows, inner = 4090, 600
    (q, s), (wq, ws) = random_q8(rows, inner, 1), random_q8(cols, inner, 2)
    q, wq, ws = aligned(q), aligned(wq), ws / (inner ** 0.5 * 40)
    for dtype in TYPES:
        check(uf, q, s, wq, ws, dtype, "silu", rand(cols, dtype=dtype, seed=3), rand(rows, cols, dtype=dtype, seed=4))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 100, 300), (5, 77, 4200), (33, 130, 4097), (40, 100, 40000), (65, 129, 127), (130, 300, 700), (700, 515, 2049)])
def test_parts(uf, shape, dtype, kind):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 5), random_q8(n, k, 6)
    ws = ws / (k ** 0.5 * 20)
    bias, residual = rand(n, dtype=dtype, seed=7), rand(m, n, dtype=dtype, seed=8)
    for b in (None, bias):
        for r in (None, residual):
            if kind is None and b is None and r is None:
                assert torch.equal(uf.matmul_q8(q, s, wq, ws, dtype=dtype, bias=None), uf.matmul_q8(q, s, wq, ws, dtype=dtype))
            else:
                check(uf, q, s, wq, ws, dtype, kind, b, r)


@pytest.mark.parametrize("shape", [(3, 50, 40), (20, 500, 4160), (200, 515, 700)])
def test_residuals_and_biases_of_other_strides(uf, shape):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 5), random_q8(n, k, 6)
    ws = ws / (k ** 0.5 * 20)
    for dtype in TYPES:
        wide, bias = rand(m, n + 9, dtype=dtype, seed=1), rand(2 * n + 1, dtype=dtype, seed=2)
        for r, b in ((wide[:, 3:3 + n], bias[1:n + 1]), (wide[:1, :n].expand(m, n), bias[1::2]), (rand(n, m, dtype=dtype, seed=3).t(), bias[:1].expand(n))):
            got = uf.matmul_q8(q, s, wq, ws, dtype=dtype, bias=b, activation="gelu", residual=r)
            assert torch.equal(got, uf.matmul_q8(q, s, wq, ws, dtype=dtype, bias=b.clone(), activation="gelu", residual=r.contiguous().clone()))
        assert (wide == rand(m, n + 9, dtype=dtype, seed=1)).all()
    # leading dimensions
    if m % 2 == 0:
        y = uf.matmul_q8(q.reshape(2, m // 2, k), s.reshape(2, m // 2), wq, ws, activation="relu", residual=torch.ones(2, m // 2, n, device="cuda"))
        assert torch.equal(y.reshape(m, n), uf.matmul_q8(q, s, wq, ws, activation="relu", residual=torch.ones(m, n, device="cuda")))


def test_activations_over_their_range(uf):
    """numbers from the smallest to the largest, infinities, NaN, through a product with one: z is the bias"""
    z = torch.cat([torch.linspace(-30, 30, 2001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30, 3e38, -3e38, 88.8, -88.8, -104.0, -200.0]),
                   torch.tensor([float("inf"), -float("inf"), float("nan")])]).cuda()
    n = z.numel()
    q, s = torch.zeros(70, 16, dtype=torch.int8, device="cuda"), torch.ones(70, device="cuda")
    wq, ws = torch.zeros(n, 16, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
    for rows in (1, 20, 70):
        for kind in KINDS[1:]:
            y = uf.matmul_q8(q[:rows], s[:rows], wq, ws, bias=z, activation=kind)
            assert torch.equal(y, y[:1].expand(rows, n)) or torch.isnan(y).any()
            y = y[-1]
            finite = torch.isfinite(z)
            want, slope = act64(z[finite].double(), kind)
            close(y[finite], want, 16 * U * z[finite].double().abs() + 2.0 ** -149)
            assert y[n - 3] == float("inf") and torch.isnan(y[n - 1])
            assert (y[z < -200] <= 0).all() if kind == "relu" else (y[(z < -200) & finite].abs() == 0).all()
            if kind == "relu":
                assert y[n - 2] == 0


def gradients(uf, x, w, bias, residual, g, kind):
    leaves = [t.requires_grad_(True) for t in (x, w, bias, residual) if t is not None]
    y = uf.linear_q8(x, w, bias=bias, activation=kind, residual=residual)
    return y, torch.autograd.grad((y,), leaves, (g,))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 17), (33, 130, 100), (129, 65, 300), (300, 257, 77), (1000, 90, 64), (2500, 530, 40)])
def test_linear(uf, dtype, kind, shape):
    m, n, k = shape
    x, w = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, residual, g = rand(n, dtype=dtype, seed=4), rand(m, n, dtype=dtype, seed=5), rand(m, n, dtype=dtype, seed=3)
    y, (dx, dw, dbias, dresidual) = gradients(uf, x, w, bias, residual, g, kind)
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    want, tolerance, slope, slope_off, corner = epilogue64(product64(q, s, wq, ws), bias.detach(), kind, residual.detach(), dtype)
    close(y, want, tolerance)
    assert torch.equal(dresidual, g)
    xr, wr, g64 = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], g.double()
    dz, dz_off = g64 * slope, g64.abs() * (slope_off + corner + U * slope.abs())
    # the scaled gradient as in the product without an epilogue
    terms = 1 if dtype == torch.bfloat16 else 2
    kept = EPS[torch.float16] ** terms + U
    left_x, left_w = (dz * ws.double()).abs().amax(1, keepdim=True), (dz * s.double()[:, None]).abs().amax(0)[:, None]
    for got, want, size, off, depth, low in (
            (dx, dz @ wr, dz.abs() @ wr.abs(), dz_off @ wr.abs(), n, left_x * wq.double().abs().sum(0)),
            (dw, dz.t() @ xr, dz.t().abs() @ xr.abs(), dz_off.t() @ xr.abs(), m, left_w * q.double().abs().sum(0))):
        close(got, want, EPS[dtype] * want.abs() + (kept + 2 * terms * depth * U) * size + off + 2.0 ** -39 * low + subnormal(dtype))
    total = dz.sum(0)
    close(dbias, total, EPS[dtype] * total.abs() + m * U * dz.abs().sum(0) + dz_off.sum(0) + subnormal(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_some_gradients_only(uf, dtype):
    m, n, k = 200, 96, 64
    x, w, bias, residual = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2), rand(n, dtype=dtype, seed=4), rand(m, n, dtype=dtype, seed=5)
    g = rand(m, n, dtype=dtype, seed=3)
    _, every = gradients(uf, x, w, bias, residual, g, "gelu")
    for i in range(4):
        one = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate((x, w, bias, residual))]
        y = uf.linear_q8(one[0], one[1], bias=one[2], activation="gelu", residual=one[3])
        assert torch.equal(torch.autograd.grad(y, one[i], g)[0], every[i])
    # without bias or residual; a bias of another type
    y = uf.linear_q8(x, w, activation="gelu")
    for a, b in zip(torch.autograd.grad(y, (x, w), g), torch.autograd.grad(uf.linear_q8(x, w, activation="gelu", residual=residual), (x, w), g)):
        assert torch.equal(a, b)
    other = bias.detach().half().requires_grad_(True)
    d, = torch.autograd.grad(uf.linear_q8(x.detach(), w.detach(), bias=other), other, g)
    assert d.dtype == torch.float16
    close(d, g.double().sum(0), EPS[torch.float16] * g.double().sum(0).abs() + m * U * g.double().abs().sum(0))
    # nothing through a relu that is closed, no infinity either
    closed = rand(n, dtype=dtype, seed=4) - 1000
    g[5, 7] = float("inf")
    _, (dx, dw, dbias) = gradients(uf, x.detach(), w.detach(), closed, None, g, "relu")
    assert (dx == 0).all() and (dw == 0).all() and (dbias == 0).all()


def test_gradients_of_other_strides(uf):
    m, n, k = 150, 100, 48
    x, w, bias, g = rand(m, k, seed=1), rand(n, k, seed=2), rand(n, seed=3), rand(m, n, seed=4)
    _, want = gradients(uf, x, w, bias, None, g, "silu")
    for other in (g.t().contiguous().t(), torch.nn.functional.pad(g, (1, 2))[:, 1:-2]):
        _, got = gradients(uf, x, w, bias, None, other, "silu")
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = rand(1, n, seed=6).expand(m, n)
    _, got = gradients(uf, x, w, bias, None, one, "silu")
    _, want = gradients(uf, x, w, bias, None, one.contiguous(), "silu")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # leading dimensions
    y, got3 = gradients(uf, x.detach().reshape(3, 50, k), w, bias, None, one.reshape(3, 50, n), "silu")
    assert y.shape == (3, 50, n) and torch.equal(got3[0].reshape(m, k), want[0]) and all(torch.equal(a, b) for a, b in zip(got3[1:], want[1:]))


def test_gradients_against_differences(uf):
    """of the formula that the forward was held to, in 64 bits, along one direction"""
    m, n, k = 40, 30, 24
    x, w, bias, residual, g = rand(m, k, seed=1), rand(n, k, seed=2, scale=0.2), rand(n, seed=3), rand(m, n, seed=4), rand(m, n, seed=5)
    for kind in KINDS:
        _, grads = gradients(uf, x, w, bias, residual, g, kind)
        (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
        at = [q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], bias.detach().double(), residual.detach().double()]
        loss = lambda v: ((act64(v[0] @ v[1].t() + v[2], kind)[0] + v[3]) * g.double()).sum().item()   # noqa: E731
        step = 1e-6
        for i in range(4):
            direction = rand(*at[i].shape, seed=9).double()
            ends = [loss([v + sign * step * direction if j == i else v for j, v in enumerate(at)]) for sign in (1, -1)]
            have = (grads[i].double() * direction).sum().item()
            size = (grads[i].double() * direction).abs().sum().item()
            assert abs(have - (ends[0] - ends[1]) / (2 * step)) <= 300 * U * size * 10 + 1e-6 * size, (kind, i)


@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_linear(uf, with_residual):
    x, gain, w, bias = (rand(100, 96, seed=1), 1 + rand(96, seed=2, scale=0.1), rand(72, 96, seed=3, scale=0.1), rand(72, seed=4))
    res = rand(100, 96, seed=5) if with_residual else None
    leaves = [t.requires_grad_(True) for t in (x, gain, w, bias) + ((res,) if with_residual else ())]
    g, h = rand(100, 72, seed=6), rand(100, 96, seed=7)
    outs = uf.norm_linear_q8(x, gain, w, residual=res, bias=bias, activation="gelu")
    got = torch.autograd.grad(outs[:1 + with_residual], leaves, (g, h)[:1 + with_residual])
    # the product alone on the norm's 8-bit rows
    q, s, total, _ = uf.rms_norm_q8(x.detach(), gain.detach(), residual=None if res is None else res.detach())
    wq, ws, _ = uf.quantize_rows(w.detach())
    assert torch.equal(outs[0], uf.matmul_q8(q, s, wq, ws, bias=bias.detach(), activation="gelu")) and torch.equal(outs[1], total)
    plain = (x, gain, w) + ((res,) if with_residual else ())
    z = product64(q, s, wq, ws) + bias.detach().double()
    dz = (g.double() * act64(z, "gelu")[1]).float()
    want = torch.autograd.grad(uf.norm_linear_q8(x, gain, w, residual=res)[:1 + with_residual], plain, (dz, h)[:1 + with_residual])
    for a, b in zip(got[:3] + got[4:], want):
        # dz is off by some 20 U of itself in either; its products by that and their own sums
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    close(got[3], dz.double().sum(0), 1e-5 * dz.double().abs().sum(0))


def test_replayed_and_on_another_stream(uf):
    x, w, bias, residual = (rand(*s, seed=i).requires_grad_(True) for i, s in enumerate(((150, 200), (300, 200), (300,), (150, 300))))
    g = rand(150, 300, seed=9)

    def step():
        y = uf.linear_q8(x, w, bias=bias, activation="gelu", residual=residual)
        return [y] + list(torch.autograd.grad(y, (x, w, bias, residual), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        [t.detach().clone() for t in step()]   # (no graph of these leaves lives while one is recorded)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        with torch.no_grad():
            x.mul_(1.25)
            bias.add_(0.1)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_no_rows_and_no_columns(uf):
    for m, n in ((0, 8), (5, 0)):
        x, w, bias = (torch.ones(*s, device="cuda", requires_grad=True) for s in ((m, 16), (n, 16), (n,)))
        residual = torch.ones(m, n, device="cuda", requires_grad=True)
        y = uf.linear_q8(x, w, bias=bias, activation="gelu", residual=residual)
        assert y.shape == (m, n)
        d = torch.autograd.grad(y.sum(), (x, w, bias, residual))
        assert [t.shape for t in d] == [t.shape for t in (x, w, bias, residual)] and all((t == 0).all() for t in d[:3])


def test_refusals(uf):
    x, w, bias, residual = rand(6, 32, seed=1), rand(20, 32, seed=2), rand(20, seed=3), rand(6, 20, seed=4)
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x), uf.quantize_rows(w)
    for bad, words in ((dict(bias=bias[:19]), "20 elements"), (dict(bias=bias[None]), "20 elements"), (dict(bias=bias.double()), "float32"),
                       (dict(bias=bias.cpu()), "GPU"), (dict(residual=residual[:5]), "shape and type"), (dict(residual=residual.half()), "shape and type"),
                       (dict(residual=residual.cpu()), "GPU"), (dict(activation="tanh"), "activation must")):
        with pytest.raises(RuntimeError, match=words):
            uf.matmul_q8(q, s, wq, ws, **bad)
        with pytest.raises(RuntimeError, match=words):
            uf.linear_q8(x, w, **bad)
    with pytest.raises(ValueError, match="no gradients"):
        uf.matmul_q8(q, s, wq, ws, bias=bias.clone().requires_grad_(True))
    x.requires_grad_(True)
    d, = torch.autograd.grad(uf.linear_q8(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(d.sum(), x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda t: uf.linear_q8(t, w, activation="relu"), (x.detach(),))


# ---------------------------------------------------------------- modules, and all of them together

def test_modules(uf):
    from geo_amd import utils_class
    torch.manual_seed(1)
    layer = utils_class.Linear_Q8(48, 20, bias=True, activation="gelu").cuda()
    with torch.no_grad():
        layer.bias.normal_()
    x, residual = rand(9, 48, seed=1), rand(9, 20, seed=2)
    y = layer(x, residual)
    y.sum().backward()
    assert layer.bias.grad.shape == (20,) and layer.weight.grad.shape == (20, 48)
    layer.eval()
    layer.prepare()
    with torch.no_grad():
        assert torch.equal(layer(x, residual), y)
    assert sorted(layer.state_dict()) == ["bias", "weight"]
    assert sorted(utils_class.Linear_Q8(4, 4).state_dict()) == ["weight"]
    gated = utils_class.GatedNormLinear_Q8(48, 20, bias=True, activation="silu", gate=0.5).cuda()
    a, total = gated(x, rand(9, 48, seed=3))
    (a.sum() + total.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in gated.parameters())
    gated.prepare()
    with torch.no_grad():
        b, same = gated(x, rand(9, 48, seed=3))
    # the normed rows are rounded to fp32 once before they come to 8 bits, or not: a number on the other side of half a step is a step
    assert torch.equal(total, same)
    assert (a - b).abs().max() <= 2 / 127 * gated.weight.abs().max() * 6


def test_teacher_keeps_its_results(uf):
    """the activation in the widening product's epilogue: the same bits as behind it, forward and backward"""
    from geo_amd import network
    for dtype in TYPES:
        torch.manual_seed(2)
        net = network.PatchMLP_q8(width=64, hidden=128, depth=2).cuda().to(dtype)
        x = torch.rand(5, 3, 32, 32).cuda().to(dtype)
        logits = net(x)
        logits.float().square().sum().backward()
        got = [p.grad.clone() for p in net.parameters()]
        for p in net.parameters():
            p.grad = None
        for layer in net.up:
            layer.activation = None
            layer.register_forward_hook(lambda m, i, out: (torch.relu(out[0]), out[1]))
        again = net(x)
        again.float().square().sum().backward()
        assert torch.equal(logits, again) and all(torch.equal(a, p.grad) for a, p in zip(got, net.parameters()))


@pytest.mark.parametrize("bits", [32, 8])
def test_gated_teacher_trains_and_serves(uf, bits):
    """the three operators as they are used: blocks with epilogues and gated norms, gradients to every parameter, the optimiser's step, and
    the prepared network"""
    from geo_amd import network
    torch.manual_seed(3)
    net = network.PatchMLP_q8(width=64, hidden=128, depth=3, activation="gelu", gated=True, bias=True).cuda()
    opt = network.AdamW(net.parameters(), lr=1e-3, state_bits=bits)
    x, target = torch.rand(8, 3, 32, 32).cuda(), torch.randint(10, (8,)).cuda()
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(3):
        opt.zero_grad()
        torch.nn.functional.cross_entropy(net(x), target).backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
        opt.step()
    assert all((a != p).any() for a, p in zip(before, net.parameters()))
    net.eval()
    with torch.no_grad():
        want = net(x)
        net.prepare()
        got = net(x)
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 0.1 * want.abs().max()


def test_command_line(uf):
    from geo_amd import main_distill
    out = main_distill.main(["--dataset", "SYNTHETIC", "--err", "5555", "--batch", "64", "--synthetic_size", "128", "--epochs", "1", "--teacher_epochs", "1",
                             "--teacher_optim", "AdamW8", "--teacher_gated", "1", "--iterations", "2"])
    assert all(math.isfinite(v) for v in out["teacher_losses"]) and math.isfinite(out["history"][0]["loss"])
