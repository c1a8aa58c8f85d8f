"""The dense 8-bit layers (rows in 8 bits, root-mean-square norm with 8-bit output, 8-bit product with its gradients) against their
formulas in 64 bits.

Tolerances follow from the formulas' roundings: U = 2^-24 is half a unit of fp32, EPS the half unit of an output's type (what
one rounding to it costs, relative); sums of n terms in fp32 are allowed n U of the sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}   # 2^-24, 2^-8, 2^-11
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
    """|got - want| <= tolerance, elementwise; NaN where NaN is wanted"""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = ((got - want).abs() > tolerance) & ~nan
    assert not bad.any(), (int(bad.sum()), ((got - want).abs() / tolerance)[bad].max().item())


def subnormal(dtype):
    """half of the smallest step of a type, below which its relative rounding does not hold"""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]


def check_rows(q, scale, n, slack=0.0):
    """q and scale of rows n in 64 bits.  fp32: the reciprocal and the product round once each (2 U of at most 127 steps)
    before the rounding to a whole number; `slack` (relative) for n itself."""
    a = n.abs().amax(-1)
    close(scale, a / 127, (3 * U + slack) * a / 127 + 2.0 ** -149)
    step = torch.where(a > 0, 127 / a, 0.0).unsqueeze(-1)
    assert ((q.double() - n * step).abs() <= 0.5 + 127 * (4 * U + 2 * slack)).all()
    assert q.abs().max() <= 127


# (rows, cols): one element, less than a chunk, odd sizes around a wave, a workgroup and the registers' limit, long rows
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 511), (1009, 513), (1, 4096), (4, 8191), (3, 16385), (2, 32768), (2, 40007)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rows(uf, dtype, shape):
    x = rand(*shape, dtype=dtype, seed=shape[1], scale=3.0)
    for out in TYPES:
        q, scale, values = uf.quantize_rows(x, values=out)
        check_rows(q, scale, x.double())
        want = q.double() * scale.double().unsqueeze(-1)
        close(values, want, (EPS[out] + U) * want.abs() + subnormal(out))
    q2, scale2, none = uf.quantize_rows(x)
    assert none is None and torch.equal(q, q2) and torch.equal(scale, scale2)


def test_rows_agree_with_elementary_operations(uf):
    """bit for bit what the same fp32 operations give one by one"""
    x = rand(257, 1111, seed=5)
    q, scale, values = uf.quantize_rows(x, values=torch.float32)
    most = x.abs().amax(-1, keepdim=True)
    want = (x * (torch.full_like(most, 127.0) / most)).round()
    assert torch.equal(q.float(), want) and torch.equal(scale, (most * (1.0 / 127.0)).squeeze(-1))
    assert torch.equal(values, want * (most * (1.0 / 127.0)))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_ties_zeros_and_values_that_are_no_numbers(uf, dtype):
    x = torch.zeros(6, 20, dtype=dtype, device="cuda")
    x[0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], dtype=dtype)      # reciprocal exactly 1: halves go to even
    x[2, 3] = float("nan")
    x[3, 5], x[3, 6] = float("inf"), 1.0
    x[4, 19] = -float("inf")
    x[5, :3] = torch.tensor([1.0, -1.0, 0.25], dtype=dtype) * (2.0 ** -120 if dtype is not torch.float16 else 2.0 ** -14)
    q, scale, values = uf.quantize_rows(x, values=torch.float32)
    assert q[0, :4].tolist() == [127, 0, 2, -2] and scale[0].item() == pytest.approx(1.0, rel=1e-6)
    assert (q[1] == 0).all() and scale[1] == 0 and (values[1] == 0).all()
    for r in (2, 3, 4):
        assert torch.isnan(scale[r]) and (q[r] == 0).all() and torch.isnan(values[r]).all()
    assert q[5, :3].tolist() == [127, -127, 32] and torch.isfinite(scale).tolist() == [True, True, False, False, False, True]


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_other_strides_and_alignments(uf, dtype):
    base = rand(40, 515, dtype=dtype, seed=3)
    for x in (base[:, 1:], base[::3, 5:260], base[:, ::2], base.t(), base[None, :7].expand(3, 7, 515), base[4], base.reshape(5, 8, 515)):
        q, scale, values = uf.quantize_rows(x, values=torch.bfloat16)
        want = uf.quantize_rows(x.contiguous().clone(), values=torch.bfloat16)
        assert q.shape == x.shape and scale.shape == x.shape[:-1] and values.shape == x.shape
        assert torch.equal(q, want[0]) and torch.equal(scale, want[1]) and torch.equal(values, want[2])


# ---------------------------------------------------------------- norm

def norm64(x, w, residual, eps):
    t = x.double() + (residual.double() if residual is not None else 0.0)
    r = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t, r, t * r * w.double()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_forward(uf, dtype, shape, with_residual):
    x, res = rand(*shape, dtype=dtype, seed=1, scale=2.0), rand(*shape, dtype=dtype, seed=2) if with_residual else None
    w = (1 + rand(shape[1], seed=3, scale=0.2)).to(dtype)
    q, scale, total, values = uf.rms_norm_q8(x, w, residual=res, eps=1e-5, values=torch.float32)
    t, r, n = norm64(x, w, res, 1e-5)
    if with_residual:
        close(total, t, (EPS[dtype] + U) * t.abs() + subnormal(dtype))
    else:
        assert total is x
    # t, t w and the sum of squares (in chains of at most cols / 64 + 64 additions) round in fp32
    check_rows(q, scale, n, slack=(shape[1] / 64 + 64) * U)
    close(values, q.double() * scale.double().unsqueeze(-1), 2 * U * values.double().abs())
    q2, scale2, total2, none = uf.rms_norm_q8(x, w, residual=res, eps=1e-5)
    assert none is None and torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(total, total2)


def norm_gradients64(t, w, eps, g, h):
    """the gradients written out, and the sums of magnitudes that bound their roundings"""
    t, w, g = t.double(), w.double(), g.double()
    r = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = g * w
    along = (u * t).mean(-1, keepdim=True)
    dx = r * (u - t * r.square() * along) + (h.double() if h is not None else 0.0)
    size = r * (u.abs() + 2 * t.abs() * r.square() * (u * t).abs().mean(-1, keepdim=True)) + (h.double().abs() if h is not None else 0.0)
    return dx, size, (g * t * r).sum(0), (g * t * r).abs().sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_backward(uf, dtype, shape, with_residual):
    rows, cols = shape
    x, w = rand(*shape, dtype=dtype, seed=1).requires_grad_(True), (1 + rand(cols, seed=3, scale=0.2)).to(dtype).requires_grad_(True)
    res = rand(*shape, dtype=dtype, seed=2).requires_grad_(True) if with_residual else None
    g, h = rand(*shape, dtype=torch.bfloat16, seed=4), rand(*shape, dtype=dtype, seed=5) if with_residual else None
    _, _, total, values = uf.rms_norm_q8(x, w, residual=res, eps=1e-5, values=torch.bfloat16)
    if with_residual:
        dx, dw, dres = torch.autograd.grad((values, total), (x, w, res), (g, h))
        assert torch.equal(dx, dres)
    else:
        dx, dw = torch.autograd.grad((values,), (x, w), (g,))
    t = x.detach().double() + (res.detach().double() if with_residual else 0.0)
    want_x, size_x, want_w, size_w = norm_gradients64(t, w.detach(), 1e-5, g, h)
    # besides the outputs' own EPS nothing is rounded below fp32: the sum is formed again, not read as it was stored
    close(dx, want_x, EPS[dtype] * want_x.abs() + (cols / 64 + 80) * U * size_x + subnormal(dtype))
    close(dw, want_w, EPS[dtype] * want_w.abs() + (rows / 64 + 80) * U * size_w + subnormal(dtype))


def test_norm_gradient_formula_against_differences():
    """central differences of the formula without the rounding to 8 bits, in 64 bits"""
    g = torch.Generator().manual_seed(0)
    t, w, gv = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 9), (9,), (3, 9)))
    dx, _, dw, _ = norm_gradients64(t, w, 1e-5, gv, None)

    def loss(t, w):
        return (t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w * gv).sum()

    step = 1e-5
    for r in range(3):
        for c in range(9):
            e = torch.zeros_like(t)
            e[r, c] = step
            assert abs((loss(t + e, w) - loss(t - e, w)) / (2 * step) - dx[r, c]) < 1e-7
    for c in range(9):
        e = torch.zeros_like(w)
        e[c] = step
        assert abs((loss(t, w + e) - loss(t, w - e)) / (2 * step) - dw[c]) < 1e-7


def test_norm_partial_gradients_and_strides(uf):
    """gradient of the sum alone, of the values alone, of a frozen weight; rows with gaps"""
    base, other = rand(33, 130, dtype=torch.bfloat16, seed=1), rand(33, 140, dtype=torch.bfloat16, seed=2)
    x, res = base[:, 1:129].requires_grad_(True), other[:, 7:135].requires_grad_(True)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    g = rand(33, 128, dtype=torch.bfloat16, seed=3)
    _, _, total, values = uf.rms_norm_q8(x, w, residual=res, values=torch.bfloat16)
    _, _, total2, values2 = uf.rms_norm_q8(x.detach().clone(), w, residual=res.detach().clone(), values=torch.bfloat16)
    assert torch.equal(total, total2) and torch.equal(values, values2)
    dx, = torch.autograd.grad((total,), (x,), (g,), retain_graph=True)
    assert torch.equal(dx, g)
    dx, = torch.autograd.grad((values,), (x,), (g,), retain_graph=True)
    want, size, _, _ = norm_gradients64(x.detach().double() + res.detach().double(), w, 1e-6, g, None)
    close(dx, want, EPS[torch.bfloat16] * want.abs() + 100 * U * size)
    with pytest.raises(ValueError, match="values"):
        uf.rms_norm_q8(x, w, residual=res)
    with torch.no_grad():
        assert uf.rms_norm_q8(x, w, residual=res)[3] is None


def test_norm_of_zeros_and_of_values_that_are_no_numbers(uf):
    x = rand(4, 64, dtype=torch.bfloat16, seed=1)
    x[1] = 0
    x[2, 7] = float("inf")
    x[3, 0] = float("nan")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, scale, _, values = uf.rms_norm_q8(x, w, values=torch.bfloat16)
    assert scale[1] == 0 and (q[1] == 0).all() and (values[1] == 0).all() and torch.isfinite(values[0]).all()
    assert torch.isnan(scale[2:]).all() and (q[2:] == 0).all() and torch.isnan(values[2:]).all()


# ---------------------------------------------------------------- product

def random_q8(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8).cuda(),
            (torch.rand(rows, generator=g) * 0.1 + 0.01).cuda())


def product64(q, s, wq, ws):
    return (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()   # sums below 2^53: exact


# rows x cols x inner: one element; every number of rows of the kernel for few rows; both tiles; cut inner dimension;
# inner dimensions that end inside a piece, a step; odd everything
PRODUCTS = [(1, 1, 1), (1, 5, 15), (2, 17, 16), (16, 64, 128), (17, 100, 200), (33, 48, 1000), (48, 4096, 513), (64, 33, 2048),
            (65, 129, 127), (100, 130, 4096), (129, 257, 129), (257, 300, 1111), (300, 40, 5000), (1, 4096, 4096),
            (2048, 6200, 160), (4000, 3100, 257), (70, 70, 13)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_product(uf, dtype, shape):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 1), random_q8(n, k, 2)
    if dtype is torch.float16:
        s = s * 0.01   # (within the type's range)
    y = uf.matmul_q8(q, s, wq, ws, dtype=dtype)
    want = product64(q, s, wq, ws)
    # the integer sum becomes a float once, two scales: three roundings, and the output's
    close(y, want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))


def test_product_of_the_largest_operands_is_exact(uf):
    """131071 products of -128 by -128 stay inside 32 bits"""
    for rows in (1, 130):
        q = torch.full((rows, 131071), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(rows, device="cuda")
        y = uf.matmul_q8(q, one, q[:1].expand(70, -1).contiguous(), torch.ones(70, device="cuda"))
        assert (y == float(131071 * 128 * 128)).all()


def test_product_of_other_strides_and_alignments(uf):
    (q, s), (wq, ws) = random_q8(150, 333, 3), random_q8(140, 333, 4)
    for m in (5, 150):
        for lo, hi in ((0, 320), (16, 333), (1, 333), (3, 259)):
            a, b = q[:m, lo:hi], wq[:, lo:hi]
            want = product64(a, s[:m], b, ws)
            close(uf.matmul_q8(a, s[:m], b, ws), want, 5 * U * want.abs())
    y = uf.matmul_q8(q[:120].reshape(4, 30, 333), s[:120].reshape(4, 30), wq, ws)
    want = product64(q[:120], s[:120], wq, ws).reshape(4, 30, 140)
    close(y, want, 5 * U * want.abs())
    x3 = rand(3, 5, 333, seed=9)
    q3, s3, _ = uf.quantize_rows(x3)     # rows with gaps behind a dimension
    want = product64(q3.reshape(15, 333), s3.reshape(15), wq, ws).reshape(3, 5, 140)
    close(uf.matmul_q8(q3, s3, wq, ws), want, 5 * U * want.abs())
    assert uf.matmul_q8(q[:0], s[:0], wq, ws).shape == (0, 140)


@pytest.mark.parametrize("m", [1, 3, 16, 17, 40, 64, 65, 200])
@pytest.mark.parametrize("lo,hi", [(0, 4099), (1, 4099), (2, 4094), (3, 4096), (0, 2051), (5, 261), (7, 700)])
def test_product_of_rows_at_odd_addresses(uf, m, lo, hi):
    """few rows and tiles, either operand alone and both, the memory's first and last bytes among them"""
    g = torch.Generator().manual_seed(7)
    q, wq = (torch.randint(-127, 128, (r, 4099), generator=g).to(torch.int8).cuda() for r in (m, 130))
    s, ws = rand(m, seed=1).abs(), rand(130, seed=2).abs()
    a, b = q[:, lo:hi], wq[:, lo:hi]
    aligned = [torch.nn.functional.pad(t, (0, -(hi - lo) % 16))[:, :hi - lo] for t in (a, b)]
    want = product64(a, s, b, ws)
    for left, right in ((a, b), (a, aligned[1]), (aligned[0], b), (a.contiguous(), b.contiguous())):
        close(uf.matmul_q8(left, s, right, ws), want, 5 * U * want.abs())


def test_product_of_rows_that_are_no_numbers(uf):
    x = rand(70, 40, seed=1)
    x[3, 4], x[66, 0] = float("nan"), float("inf")
    x[5] = 0
    w = rand(20, 40, seed=2)
    q, s, _ = uf.quantize_rows(x)
    wq, ws, _ = uf.quantize_rows(w)
    for rows in (slice(0, 8), slice(0, 70)):
        y = uf.matmul_q8(q[rows], s[rows], wq, ws)
        bad = torch.isnan(s[rows])
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all() and (y[5] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 7), (1, 70, 200), (65, 129, 127), (257, 300, 130), (700, 64, 48), (48, 1000, 333),
                                   (1500, 3100, 4000)])
def test_linear(uf, dtype, shape):
    """forward and both gradients of linear_q8 against the product of the rounded operands in 64 bits"""
    m, n, k = shape
    x, w = rand(m, k, dtype=dtype, seed=1).requires_grad_(True), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5).requires_grad_(True)
    g = rand(m, n, dtype=dtype, seed=3)
    y = uf.linear_q8(x, w)
    dx, dw = torch.autograd.grad((y,), (x, w), (g,))
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    want = product64(q, s, wq, ws)
    close(y, want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))
    xr, wr, g64 = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], g.double()
    # the scaled gradient: one fp16 number (EPS) or two (EPS^2), the last one's steps 2^-39 of the row's largest; fp32 sums of all terms
    terms = 1 if dtype == torch.bfloat16 else 2
    kept = EPS[torch.float16] ** terms + U
    left_x, left_w = (g64 * ws.double()).abs().amax(1, keepdim=True), (g64 * s.double()[:, None]).abs().amax(0)[:, None]
    for got, want, size, depth, low in ((dx, g64 @ wr, g64.abs() @ wr.abs(), n, left_x * wq.double().abs().sum(0)),
                                        (dw, g64.t() @ xr, g64.t().abs() @ xr.abs(), m, left_w * q.double().abs().sum(0))):
        close(got, want, EPS[dtype] * want.abs() + (kept + 2 * terms * depth * U) * size + 2.0 ** -39 * low + subnormal(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_rows_of_any_magnitude(uf, dtype):
    """a row of a gradient is as exact whatever its magnitude; zeros stay zeros, infinities and NaN stay in their row and column"""
    m, n, k = 150, 90, 70
    x, w, g = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2), rand(m, n, dtype=dtype, seed=3)
    g = (g.double() * 2.0 ** ((torch.arange(m, device="cuda") * 37 % 181) - 90).double()[:, None]).to(dtype)
    g[7], g[20, 5], g[40, 60], g[130, 5] = 0, float("inf"), float("nan"), -float("inf")
    dx, dw = torch.autograd.grad((uf.linear_q8(x.requires_grad_(True), w.requires_grad_(True)),), (x, w), (g,))
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    xr, wr, g64 = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], g.double()
    bad_rows, bad_cols = ~torch.isfinite(g64).all(1), ~torch.isfinite(g64).all(0)
    assert not torch.isfinite(dx[bad_rows]).any() and not torch.isfinite(dw[bad_cols]).any() and (dx[7] == 0).all()
    terms = 1 if dtype == torch.bfloat16 else 2
    kept = EPS[torch.float16] ** terms + U
    a, b = g64[~bad_rows], g64[:, ~bad_cols].t()
    low = 2.0 ** -39 * (a * ws.double()).abs().amax(1, keepdim=True) * wq.double().abs().sum(0)
    close(dx[~bad_rows], a @ wr, EPS[dtype] * (a @ wr).abs() + (kept + 2 * terms * n * U) * (a.abs() @ wr.abs()) + low + subnormal(dtype))
    low = 2.0 ** -39 * (b * s.double()).abs().amax(1, keepdim=True) * q.double().abs().sum(0)
    close(dw[~bad_cols], b @ xr, EPS[dtype] * (b @ xr).abs() + (kept + 2 * terms * m * U) * (b.abs() @ xr.abs()) + low + subnormal(dtype))


@pytest.mark.parametrize("shape", [(70000, 33, 20), (33, 20011, 20), (5000, 1100, 40)])
def test_gradients_of_long_sides(uf, shape):
    """maxima joined from many blocks of the gradient, the largest element anywhere"""
    m, n, k = shape
    x, w, g = rand(m, k, seed=1), rand(n, k, seed=2), rand(m, n, seed=3)
    rows, cols = torch.arange(0, m, 97, device="cuda"), torch.arange(0, n, 31, device="cuda")
    g[rows, rows * 13 % n] = 2.0 ** 40
    g[cols * 29 % m, cols] = -2.0 ** 50
    dx, dw = torch.autograd.grad((uf.linear_q8(x.requires_grad_(True), w.requires_grad_(True)),), (x, w), (g,))
    (q, s, _), (wq, ws, _) = uf.quantize_rows(x.detach()), uf.quantize_rows(w.detach())
    xr, wr, g64 = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None], g.double()
    kept = EPS[torch.float16] ** 2 + U
    low = 2.0 ** -39 * (g64 * ws.double()).abs().amax(1, keepdim=True) * wq.double().abs().sum(0)
    close(dx, g64 @ wr, U * (g64 @ wr).abs() + (kept + 4 * n * U) * (g64.abs() @ wr.abs()) + low)
    low = 2.0 ** -39 * (g64 * s.double()[:, None]).abs().amax(0)[:, None] * q.double().abs().sum(0)
    close(dw, g64.t() @ xr, U * (g64.t() @ xr).abs() + (kept + 4 * m * U) * (g64.t().abs() @ xr.abs()) + low)


def test_linear_needs_one_gradient_only(uf):
    x, w, g = rand(100, 96, seed=1), rand(72, 96, seed=2), rand(100, 72, seed=3)
    both = torch.autograd.grad(uf.linear_q8(x.requires_grad_(True), w.requires_grad_(True)), (x, w), g)
    only_x, = torch.autograd.grad(uf.linear_q8(x, w.detach()), (x,), g)
    only_w, = torch.autograd.grad(uf.linear_q8(x.detach(), w), (w,), g)
    assert torch.equal(both[0], only_x) and torch.equal(both[1], only_w)
    # an upstream gradient of other strides, a constant one of stride 0
    y = uf.linear_q8(x, w)
    turned, = torch.autograd.grad(y, (x,), g.t().contiguous().t(), retain_graph=True)
    assert torch.equal(turned, both[0])
    y.sum().backward()
    ones, = torch.autograd.grad(uf.linear_q8(x, w), (x,), torch.ones_like(g))
    assert torch.equal(x.grad, ones)


@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_linear_is_the_norm_and_the_product(uf, with_residual):
    x, gain, w = (rand(3, 50, 96, seed=1).requires_grad_(True), (1 + rand(96, seed=2, scale=0.1)).requires_grad_(True),
                  rand(72, 96, seed=3).requires_grad_(True))
    res = rand(3, 50, 96, seed=4).requires_grad_(True) if with_residual else None
    y, total = uf.norm_linear_q8(x, gain, w, residual=res)
    with torch.no_grad():
        q, s, t, _ = uf.rms_norm_q8(x, gain, residual=res)
        wq, ws, _ = uf.quantize_rows(w)
        assert torch.equal(y, uf.matmul_q8(q, s, wq, ws)) and torch.equal(total, t)
    gy, gt = rand(3, 50, 72, seed=5), rand(3, 50, 96, seed=6)
    inputs = (x, gain, w) + ((res,) if with_residual else ())
    outs, grads = ((y, total), (gy, gt)) if with_residual else ((y,), (gy,))
    got = torch.autograd.grad(outs, inputs, grads)
    xr, wr = q.double() * s.double()[..., None], wq.double() * ws.double()[:, None]
    dn = gy.double() @ wr
    want_x, size_x, want_gain, size_gain = norm_gradients64(t.detach().reshape(150, 96), gain.detach(), 1e-6, dn.reshape(150, 96),
                                                            gt.reshape(150, 96) if with_residual else None)
    close(got[0].reshape(150, 96), want_x, 1e-4 * size_x + 1e-6)
    close(got[1], want_gain, 1e-4 * size_gain)
    close(got[2], gy.double().reshape(150, 72).t() @ xr.reshape(150, 96), 1e-4 * (gy.double().abs().reshape(150, 72).t() @ xr.abs().reshape(150, 96)))
    if with_residual:
        assert torch.equal(got[0], got[3])


# ---------------------------------------------------------------- all of them

def test_on_another_stream_and_in_a_graph(uf):
    """the operators run on the current stream, and a captured graph of them gives the eager results on every replay"""
    x, res, gain, w = rand(9, 256, dtype=torch.bfloat16, seed=1), rand(9, 256, dtype=torch.bfloat16, seed=2), torch.ones(
        256, dtype=torch.bfloat16, device="cuda"), rand(320, 256, seed=3)
    wq, ws, _ = uf.quantize_rows(w)

    def step():
        q, s, total, _ = uf.rms_norm_q8(x, gain, residual=res)
        return uf.matmul_q8(q, s, wq, ws, dtype=torch.bfloat16), total

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        x.copy_(rand(9, 256, dtype=torch.bfloat16, seed=10 + seed))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_same_results_on_every_run(uf):
    x, w = rand(500, 1000, dtype=torch.bfloat16, seed=1).requires_grad_(True), rand(300, 1000, dtype=torch.bfloat16, seed=2).requires_grad_(True)
    g, gain = rand(500, 300, dtype=torch.bfloat16, seed=3), torch.ones(1000, dtype=torch.bfloat16, device="cuda", requires_grad=True)

    def run():
        y, _ = uf.norm_linear_q8(x, gain, w)
        return torch.autograd.grad(y, (x, gain, w), g)

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_no_rows(uf):
    x, w = torch.empty(0, 24, device="cuda", requires_grad=True), rand(10, 24).requires_grad_(True)
    gain = torch.ones(24, device="cuda", requires_grad=True)
    q, s, values = uf.quantize_rows(x.detach(), values=torch.bfloat16)
    assert q.shape == (0, 24) and s.shape == (0,) and values.shape == (0, 24)
    y = uf.linear_q8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 10, device="cuda"))
    assert y.shape == (0, 10) and dx.shape == (0, 24) and (dw == 0).all()
    _, _, total, values = uf.rms_norm_q8(x, gain, residual=x.detach(), values=torch.float32)
    dx, dgain = torch.autograd.grad(values, (x, gain), torch.empty(0, 24, device="cuda"))
    assert dx.shape == (0, 24) and (dgain == 0).all()
    y, total = uf.norm_linear_q8(x, gain, w, residual=x.detach())
    assert y.shape == (0, 10) and total.shape == (0, 24)


def test_offsets_beyond_32_bits(uf):
    """matrices of more than 2^32 bytes (and 2^31 elements): their last rows against the same rows by themselves"""
    rows, cols = 70001, 33000
    x = torch.randn(rows, 1, generator=torch.Generator().manual_seed(1)).cuda().bfloat16() * torch.linspace(-1, 1, cols, device="cuda").bfloat16()
    w = torch.ones(cols, dtype=torch.bfloat16, device="cuda")
    last = x[-3:].clone()
    q, s, values = uf.quantize_rows(x, values=torch.bfloat16)
    want = uf.quantize_rows(last, values=torch.bfloat16)
    assert torch.equal(q[-3:], want[0]) and torch.equal(s[-3:], want[1]) and torch.equal(values[-3:], want[2])
    del q, values
    q, s, total, _ = uf.rms_norm_q8(x, w, residual=x)
    want = uf.rms_norm_q8(last, w, residual=last)
    assert torch.equal(q[-3:], want[0]) and torch.equal(s[-3:], want[1]) and torch.equal(total[-3:], want[2])
    del total
    wq, ws = random_q8(40, cols, 5)
    y = uf.matmul_q8(q, s, wq, ws)                       # a left operand of more than 2^31 bytes
    want = product64(q[-3:], s[-3:], wq, ws)
    close(y[-3:], want, 5 * U * want.abs())
    del q, x, y
    (q, s), (wq, ws) = random_q8(rows, 64, 6), random_q8(cols, 64, 7)
    y = uf.matmul_q8(q, s, wq, ws, dtype=torch.bfloat16)  # a result of more than 2^31 elements
    want = product64(q[-3:], s[-3:], wq, ws)
    close(y[-3:], want, (EPS[torch.bfloat16] + 4 * U) * want.abs())


def test_refusals(uf):
    x, w = rand(4, 16), rand(8, 16)
    q, s, _ = uf.quantize_rows(x)
    wq, ws, _ = uf.quantize_rows(w)
    bad = [lambda: uf.quantize_rows(x.double()), lambda: uf.quantize_rows(x.cpu()), lambda: uf.quantize_rows(x[:, :0]),
           lambda: uf.quantize_rows(x, values=torch.int8),
           lambda: uf.rms_norm_q8(x, w[0, :8]), lambda: uf.rms_norm_q8(x, w[0].bfloat16()), lambda: uf.rms_norm_q8(x, w[0], residual=x[:2]),
           lambda: uf.rms_norm_q8(x, w[0], residual=x.half()), lambda: uf.rms_norm_q8(x, w[0], eps=-1.0),
           lambda: uf.rms_norm_q8(x, w[0].cpu()),
           lambda: uf.matmul_q8(q, s, wq[:, :8], ws), lambda: uf.matmul_q8(x, s, wq, ws), lambda: uf.matmul_q8(q, s[:2], wq, ws),
           lambda: uf.matmul_q8(q, s.double(), wq, ws), lambda: uf.matmul_q8(q, s, wq, ws, dtype=torch.int32),
           lambda: uf.matmul_q8(q, s, wq.cpu(), ws), lambda: uf.matmul_q8(q, s, wq[None], ws),
           lambda: uf.matmul_q8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s[:1],
                                torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), ws[:1]),
           lambda: uf.linear_q8(x, w[:, :3])]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")
