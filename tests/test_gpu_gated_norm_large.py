"""The gated norm where rows are many: two at once in 16 bits over several waves with an odd last one, units of several rows with runs that end
inside them, outputs past the caches, and such rows beyond the range of squares or without numbers, against the formulas in 64 bits."""
import pytest
import torch

from tests.test_gpu_gated_norm import EPS, TINY, U, call, check, close, formulas, inputs, leaves, rand, uf  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# rows (odd: the last of two is computed twice and stored once), columns, runs of rows that share a gate.  Two, three and four waves for a row; three,
# nine and sixteen to seventeen rows in a unit; runs of a unit's rows, of fewer and of many, ends inside units and at their borders; the
# last: outputs of more than 128 MB, and 9.2 M elements in rows at odd places
CASES = [(2049, 1100, 683), (2049, 1100, 3), (4097, 2056, 241), (4097, 2056, 17), (4097, 2056, 1), (8191, 4096, 1), (8190, 4096, 13),
         (8193, 4096, 2731), (8193, 4096, 3), (2051, 4481, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_both_passes(uf, case, dtype):
    rows, cols, runs = case
    check(uf, inputs(rows, cols, dtype, runs=runs, seed=runs))


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("parts", [(False, False, None), (True, False, 3), (False, True, 3), (True, True, None)])
def test_parts_that_are_not_there(uf, parts, dtype):
    post, scale, runs = parts
    check(uf, inputs(2049, 1100, dtype, runs=runs, post=post, scale=scale))
    check(uf, inputs(2049, 1100, dtype, runs=runs, post=post, scale=scale), want_h=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(2049, 1100, 3), (4097, 2056, 1), (8193, 4096, 3)])
def test_eight_bits(uf, case, dtype):
    rows, cols, runs = case
    v = inputs(rows, cols, dtype, runs=runs)
    for eight in TYPES:
        with torch.no_grad():
            q, scale, total, values = call(uf, v, 1e-5, eight)
            assert torch.equal(total, call(uf, v, 1e-5)[1])
        scale = scale.reshape(-1)
        n, off = formulas({k: t.float() if t is not None else None for k, t in v.items()}, 1e-5)["out"]
        a = n.abs().amax(-1)
        slack = (off / a[:, None]).amax(-1)
        assert ((scale.double() - a / 127).abs() <= (slack + 4 * U) * a / 127).all()
        assert ((q.double() - n * (127 / a)[:, None]).abs() <= 0.5 + 127 * (4 * U + 2 * slack[:, None])).all()
        want = q.double() * scale.double()[:, None]
        close(values, want, (EPS[eight] + U) * want.abs() + TINY[eight])


@pytest.mark.parametrize("case", [(2049, 1100), (4097, 2056), (8193, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_beyond_the_range_of_squares(uf, case, dtype):
    """the first, the second or both of two rows at once, in either norm or both; the last row of an odd count"""
    rows, cols = case
    for size in (1e25, 1e-25):
        v = inputs(rows, cols, dtype, runs=1, post=size > 1)   # (beside a tiny residual the normed branch would hide it)
        x_size, residual_size = torch.ones(rows, 1, device="cuda"), torch.ones(rows, 1, device="cuda")
        for row in (0, 3, 6, 7, 100, 131, 256, rows - 1):
            x_size[row] = size
        for row in (0, 2, 5, 6, 7, 101, 256, 257, rows - 1):
            residual_size[row] = size
        if size < 1:   # one of both would be all of the sum
            residual_size = x_size
        v["x"], v["residual"] = (v["x"] * x_size.to(dtype)), (v["residual"] * residual_size.to(dtype))
        g = rand(rows, cols, dtype=dtype, seed=5, scale=1e-3)
        if size > 1:
            check(uf, v, eps=0.0, g=g, h=g)
        else:   # gradients of such rows pass the range themselves
            with torch.no_grad():
                got = call(uf, v, 0.0)
            want = formulas(v, 0.0)
            close(got[0], *want["out"])
            close(got[1], *want["total"])
        with torch.no_grad():
            q, scale, _, values = call(uf, v, 0.0, torch.float32)
        n, off = formulas({k: t.float() if t is not None else None for k, t in v.items()}, 0.0)["out"]
        most = n.abs().amax(-1, keepdim=True)
        assert ((values.double() - n).abs() <= most / 127 * 0.5 + 2 * off + 4 * U * most).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(2049, 1100), (4097, 2056)])
def test_rows_that_hold_no_numbers(uf, case, dtype):
    """stay by themselves, whichever of two at once they are"""
    rows, cols = case
    v = inputs(rows, cols, dtype, runs=1)
    with torch.no_grad():
        good = call(uf, v, 1e-6), call(uf, v, 1e-6, torch.float32)
        bad = {1: ("x", float("nan")), 4: ("residual", float("inf")), 6: ("x", -float("inf")), 7: ("residual", float("nan")), rows - 1: ("x", float("nan"))}
        for row, (k, value) in bad.items():
            v[k][row, cols - 1] = value
        v["x"][9], v["residual"][9] = 0.0, 0.0
        out, total = call(uf, v, 1e-6)
        q, scale, total8, values = call(uf, v, 1e-6, torch.float32)
    sound = torch.ones(rows, dtype=torch.bool, device="cuda")
    sound[list(bad) + [9]] = False
    assert torch.equal(out[sound], good[0][0][sound]) and torch.equal(total[sound], good[0][1][sound])
    assert torch.equal(q[sound], good[1][0][sound]) and torch.equal(values[sound], good[1][3][sound]) and torch.equal(total8[sound], good[1][2][sound])
    assert torch.isnan(out[list(bad), cols - 1]).all() and torch.isnan(scale[list(bad)]).all() and (q[list(bad)] == 0).all()
    assert (out[9] == 0).all() and (total[9] == 0).all() and (values[9] == 0).all() and scale[9] == 0


@pytest.mark.parametrize("dtype", TYPES[:2])
def test_same_bits_on_every_run(uf, dtype):
    v = inputs(8193, 4096, dtype, runs=3)
    first = check(uf, v)
    for _ in range(3):
        again = check(uf, v)
        assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignments(uf, dtype):
    """many rows at odd addresses, which are read through the caches: the same bits"""
    rows, cols = 4097, 2056
    base = inputs(rows, cols, dtype, runs=17)
    want = check(uf, base)
    v = leaves(base)
    for k in ("x", "residual"):
        wide = torch.full((rows, cols + 3), 9.0, dtype=dtype, device="cuda")
        wide[:, 1:1 + cols] = base[k]
        v[k] = wide[:, 1:1 + cols].detach().requires_grad_(True)
    g, h = rand(rows, cols, dtype=dtype, seed=77), rand(rows, cols, dtype=dtype, seed=78)
    # (gates per run take x of three dimensions, which odd distances do not have: a gate of every row instead)
    every = base["gate"].repeat_interleave(rows // 17, 0).requires_grad_(True)
    out, total = uf.gated_norm(v["x"], v["residual"], v["weight"], v["post"], every, v["scale"], 1e-5)
    assert torch.equal(out, want["out"]) and torch.equal(total, want["total"])
    names = ["x", "residual", "weight", "post", "scale"]
    for name, d in zip(names, torch.autograd.grad((out, total), [v[k] for k in names], (g, h))):
        tolerance = formulas(base, 1e-5, g, h)["d" + name][1]
        if name in ("x", "residual"):
            assert torch.equal(d, want["d" + name]), name
        else:   # sums over rows, by other runs
            assert ((d.double() - want["d" + name].double()).abs() <= 2 * tolerance).all(), name
