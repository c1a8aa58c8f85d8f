"""Calls on a stream that is not the current one: their scratch and results are memory of the current stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from geo_amd import capi
    return capi


@pytest.mark.parametrize("call", ["forward", "values", "quantize"])
def test_result_and_scratch_of_a_call_on_another_stream(capi, call):
    """The result is whole where it is used next, and scratch handed out again is not written over while the call needs it,
    also where the given stream is far behind."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.rand((16, 32, 16, 16), generator=g).cuda(), (torch.rand((32, 32, 3, 3), generator=g) - 0.5).cuda()
    d = capi.make_desc(x.shape, w.shape, 64, (1, 1))
    run = {"forward": lambda s: capi.conv2d_add_partial_forward(x, w, 64, (1, 1), stream=s),
           "values": lambda s: capi.conv2d_add_partial_values(x, w, d, 64, stream=s),
           "quantize": lambda s: capi.quantize(x, 4, stream=s)}[call]
    ref = run(None)
    side = torch.cuda.Stream()
    for _ in range(3):
        # (memory that the next result may get holds something else)
        torch.full_like(ref, -7)
        with torch.cuda.stream(side):
            for _ in range(20):
                torch.rand(4096, 4096, device="cuda").sort()
        y = run(side)
        over = torch.full((capi.workspace_size(d),), 255, dtype=torch.uint8, device="cuda")
        assert torch.equal(y, ref)
        del over, y
    torch.cuda.synchronize()
