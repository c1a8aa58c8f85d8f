"""Calls on given streams run beside each other: a call waits for nothing but its own stream, and the current stream only for
results that were allocated for it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from geo_amd import capi
    return capi


@pytest.fixture(scope="module")
def layer(capi):
    g = torch.Generator().manual_seed(5)
    x, w = torch.rand((16, 32, 16, 16), generator=g).cuda(), (torch.rand((32, 32, 3, 3), generator=g) - 0.5).cuda()
    ref = capi.conv2d_add_partial_forward(x, w, 64, (1, 1))
    capi.quantize(x, 4)
    torch.rand(2 ** 24, device="cuda").sort()
    torch.cuda.synchronize()
    return x, w, ref


def busy(stream, sorts=150):
    """long work on a stream (a tenth of a second and more); the event behind it"""
    with torch.cuda.stream(stream):
        for _ in range(sorts):
            torch.rand(2 ** 24, device="cuda").sort()
        return stream.record_event()


def test_two_calls_on_two_streams_overlap(capi, layer):
    """of several streams (some may share a hardware queue with the busy one) one is done while the other still works"""
    x, w, ref = layer
    others = [torch.cuda.Stream() for _ in range(4)]
    first = torch.cuda.Stream()
    for s in others:   # (memory of their own, before anything is timed)
        capi.conv2d_add_partial_forward(x, w, 64, (1, 1), stream=s)
    torch.cuda.synchronize()
    behind = busy(first)
    y = capi.conv2d_add_partial_forward(x, w, 64, (1, 1), stream=first)
    results, early = [], False
    for s in others:
        results.append(capi.conv2d_add_partial_forward(x, w, 64, (1, 1), stream=s))
    done = [s.record_event() for s in others]
    while not behind.query():
        early = early or any(e.query() for e in done)
        if early:
            break
    assert early
    for r in results + [y]:
        assert torch.equal(r, ref)


@pytest.mark.parametrize("given", ["out", "out and workspace"])
def test_results_in_the_callers_memory_hold_up_nobody(capi, layer, given):
    """of several streams (one may share the current one's hardware queue) there is one that the current stream passes by"""
    x, w, ref = layer
    d = capi.make_desc(x.shape, w.shape, 64, (1, 1))
    passed = False
    for side in [torch.cuda.Stream() for _ in range(4)]:
        out, q = torch.empty_like(ref), torch.empty_like(x)
        ws = torch.empty(capi.workspace_size(d), dtype=torch.uint8, device="cuda") if given != "out" else None
        torch.cuda.synchronize()
        behind = busy(side)
        capi.conv2d_add_partial_forward(x, w, 64, (1, 1), out=out, workspace=ws, stream=side)
        capi.quantize(x, 4, out=q, stream=side)
        torch.cuda.current_stream().record_event().synchronize()
        passed = passed or not behind.query()
        side.synchronize()
        assert torch.equal(out, ref) and torch.equal(q, capi.quantize(x, 4))
    assert passed


def test_a_result_lives_until_the_current_stream_has_read_it(capi, layer):
    """freed while the current stream is behind, its memory goes to no call on the stream that it came from"""
    x, w, ref = layer
    side, other = torch.cuda.Stream(), torch.zeros_like(x)
    for _ in range(3):
        y = capi.conv2d_add_partial_forward(x, w, 64, (1, 1), stream=side)
        busy(torch.cuda.current_stream(), 20)
        kept = y.clone()
        del y
        more = [capi.conv2d_add_partial_forward(other, w, 64, (1, 1), out=None, stream=s) for s in (side, side)]
        assert torch.equal(kept, ref)
        del more
    torch.cuda.synchronize()


def test_converted_operands_are_in_the_calls_order(capi, layer):
    """operands of other types and strides are converted on the given stream, which may be far behind"""
    x, w, ref = layer
    w_n, b_n = torch.linspace(0.5, 2, 32, device="cuda", dtype=torch.float64), torch.linspace(-1, 1, 64, device="cuda")[::2]
    want, _ = capi.layer_epilogue(ref, 64, w_n, b_n)
    side = torch.cuda.Stream()
    for _ in range(3):
        busy(side, 20)
        got, _ = capi.layer_epilogue(ref, 64, w_n, b_n, stream=side)
        over = [torch.full((32,), float("nan"), device="cuda") for _ in range(8)]
        assert torch.equal(got, want)
        del over
