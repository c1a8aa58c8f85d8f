"""Every kernel of the 8-bit product, at shapes that tests/test_dense_plan.py holds to it."""
import pytest
import torch

from tests.test_dense_plan import SHAPES, STREAMED, TILES
from tests.test_gpu_dense import EPS, TYPES, U, close, product64, random_q8, subnormal, uf  # noqa: F401

pytestmark = pytest.mark.gpu


def aligned(t):
    return torch.nn.functional.pad(t, (0, -t.shape[1] % 16))[:, :t.shape[1]]


def check(uf, q, s, wq, ws, dtype):
    y = uf.matmul_q8(q, s, wq, ws, dtype=dtype)
    want = product64(q, s, wq, ws)
    close(y, want, (EPS[dtype] + 4 * U) * want.abs() + subnormal(dtype))   # as test_product: three roundings and the output's


@pytest.mark.parametrize("shape", SHAPES)
def test_kernels(uf, shape):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k, 1), random_q8(n, k, 2)
    q, wq = aligned(q), aligned(wq)
    for dtype in TYPES if SHAPES[shape][0] == STREAMED else [TYPES[k % 3]]:
        check(uf, q, s * 0.01 if dtype is torch.float16 else s, wq, ws, dtype)


@pytest.mark.parametrize("shape", [s for s in SHAPES if SHAPES[s][0] == STREAMED])
def test_streamed_rows_with_gaps_and_no_numbers(uf, shape):
    """operands inside wider matrices; a row whose scale is NaN, rows and columns of zeros"""
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k + 64, 3), random_q8(n, k + 64, 4)
    q, wq = aligned(q)[:, 16:16 + k], aligned(wq)[:, 32:32 + k]
    s, ws = s.clone(), ws.clone()
    s[1], s[2], ws[n // 2], ws[n - 1] = float("nan"), 0, 0, float("nan")
    check(uf, q, s, wq, ws, torch.float32)


@pytest.mark.parametrize("shape", [s for s in SHAPES if SHAPES[s][0] == TILES and s[0] * s[1] * s[2] < 4e10])
def test_tiles_of_rows_at_odd_addresses(uf, shape):
    m, n, k = shape
    (q, s), (wq, ws) = random_q8(m, k + 1, 5), random_q8(n, k + 1, 6)
    check(uf, q[:, 1:], s, wq[:, :k], ws, torch.float32)
    check(uf, aligned(q)[:, :k], s, wq[:, 1:], ws, torch.bfloat16)
