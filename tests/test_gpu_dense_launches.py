"""More rows, or columns, than the threads of one launch reach: a launch counts them in 32 bits, and what passes that would be left as
the allocator handed it out.  One wave serves four rows of a narrow matrix, a workgroup of 512 threads 16 columns of a product."""
import pytest
import torch

from tests.test_gpu_dense import U, close, product64, uf  # noqa: F401

pytestmark = pytest.mark.gpu

ROWS = 2 ** 28 + 1024   # 2^32 threads and some more; whole periods of 64


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def periodic(t):
    """every row is what the first ones are, which other tests look at"""
    t = t.view(-1, 64)
    return bool((t == t[:1]).all())


def all_are(t, value):   # (a comparison in an assert would be shown, element by element, should it fail)
    return bool((t == value).all())


def test_rows_of_one_column(uf):
    x = (1 + torch.arange(64, device="cuda", dtype=torch.bfloat16)).repeat(ROWS // 64)[:, None]
    q, scale, values = uf.quantize_rows(x, values=torch.bfloat16)
    assert all_are(q, 127) and periodic(scale) and all_are(values, x)
    close(scale[:64], x[:64, 0].double() / 127, 3 * U * x[:64, 0].double() / 127)
    del q, scale, values
    one = torch.ones(1, dtype=torch.bfloat16, device="cuda")
    q, scale, total, values = uf.rms_norm_q8(x, one, residual=x, eps=0.0, values=torch.bfloat16)
    assert all_are(q, 127) and periodic(scale) and all_are(total, 2 * x) and all_are(values, 1)


def test_loss_of_two_columns(uf):
    v = torch.linspace(-3, 3, 64, device="cuda").bfloat16()
    z = torch.stack((torch.zeros_like(v), v), 1).repeat(ROWS // 64, 1)
    t, index = torch.zeros(1, 1, device="cuda").expand(ROWS, 1), torch.ones(1, 1, dtype=torch.int32, device="cuda").expand(ROWS, 1)
    z = z.requires_grad_(True)
    loss = uf.distill_topk(z, t, index, reduction="none")
    assert periodic(loss.detach())
    close(loss[:64], torch.log1p(torch.exp(-v.double())), 64 * 8 * U * torch.ones(64, device="cuda"))
    dz, = torch.autograd.grad(loss, z, torch.ones(1, device="cuda").expand(ROWS))
    assert periodic(dz[:, 0].contiguous()) and periodic(dz[:, 1].contiguous())


def test_product_of_many_columns(uf):
    cols = 2 ** 27 + 4000
    g = torch.Generator("cuda").manual_seed(1)
    wq = torch.randint(-127, 128, (cols, 16), generator=g, dtype=torch.int8, device="cuda")
    ws = torch.rand(cols, generator=g, device="cuda")
    q, s = wq[5:8].clone(), ws[5:8].clone()
    y = uf.matmul_q8(q, s, wq, ws, dtype=torch.bfloat16)
    for at in (slice(0, 5000), slice(2 ** 26, 2 ** 26 + 5000), slice(2 ** 27 - 100, cols)):
        want = product64(q, s, wq[at], ws[at])
        close(y[:, at], want, (2.0 ** -8 + 5 * U) * want.abs())
