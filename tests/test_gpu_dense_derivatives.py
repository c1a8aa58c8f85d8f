"""What the dense operators and the loss have no rule for is refused, not answered with something else: forward-mode tangents, second
derivatives, recording of the calls as operations."""
import pytest
import torch
from torch.autograd import forward_ad

from tests.test_gpu_dense import rand, uf  # noqa: F401

pytestmark = pytest.mark.gpu


def operands():
    g = torch.Generator().manual_seed(7)
    index = torch.stack([torch.randperm(24, generator=g)[:5] for _ in range(12)]).cuda()
    return dict(x=rand(12, 24, seed=1), gain=1 + rand(24, seed=2, scale=0.1), w=rand(16, 24, seed=3), residual=rand(12, 24, seed=4), t=rand(12, 5, seed=5),
                index=index)


CALLS = {"linear": lambda uf, o: uf.linear_q8(o["x"], o["w"]),
         "norm_linear": lambda uf, o: uf.norm_linear_q8(o["x"], o["gain"], o["w"], residual=o["residual"])[0],
         "norm": lambda uf, o: uf.rms_norm_q8(o["x"], o["gain"], residual=o["residual"], values=torch.float32)[3],
         "loss": lambda uf, o: uf.distill_topk(o["x"], o["t"], o["index"])}


@pytest.mark.parametrize("call", list(CALLS) + ["rows", "product"])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents_are_refused(uf, call, grad_mode):
    """a tangent that is dropped would be a derivative of zero"""
    o = operands()
    q, s, _ = uf.quantize_rows(o["x"])
    wq, ws, _ = uf.quantize_rows(o["w"])
    run = {**CALLS, "rows": lambda uf, o: uf.quantize_rows(o["x"], values=torch.float32)[2],
           "product": lambda uf, o: uf.matmul_q8(q, o["s"], wq, ws)}[call]
    o["s"] = s
    run(uf, o)
    for name in ("x", "gain", "w", "residual", "t", "s"):
        used = {"linear": "xw", "rows": "x", "product": "s", "loss": "xt"}.get(call, ["x", "gain", "residual"] + ["w"] * (call == "norm_linear"))
        if name not in used:
            continue
        with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
            dual = dict(o, **{name: forward_ad.make_dual(o[name], torch.ones_like(o[name]))})
            with pytest.raises(RuntimeError, match="tangent|jvp"):
                run(uf, dual)


@pytest.mark.parametrize("call", list(CALLS))
def test_second_derivatives_are_refused(uf, call):
    """a penalty on a gradient would add nothing to the result"""
    for name in {"linear": "xw", "loss": "x"}.get(call, ("x", "gain", "residual") + ("w",) * (call == "norm_linear")):
        o = operands()
        o[name].requires_grad_(True)
        first, = torch.autograd.grad(CALLS[call](uf, o).sum(), o[name])
        again, = torch.autograd.grad(CALLS[call](uf, o).sum(), o[name], create_graph=True)
        assert torch.equal(first, again.detach()) and again.requires_grad   # asked for and not used: the value is there
        with pytest.raises(RuntimeError, match="once only"):
            again.square().sum().backward()
        # beside a term that has a second derivative too
        total = CALLS[call](uf, o).sum() + o[name].pow(3).sum()
        both, = torch.autograd.grad(total, o[name], create_graph=True)
        with pytest.raises(RuntimeError, match="once only"):
            torch.autograd.grad(both.sum(), o[name])


def test_gradient_of_the_sum_alone_has_a_second_derivative(uf):
    """what passes by the norm, x + residual, is linear"""
    o = operands()
    x = o["x"].requires_grad_(True)
    _, _, total, _ = uf.rms_norm_q8(x, o["gain"], residual=o["residual"], values=torch.float32)
    g, = torch.autograd.grad(total.pow(3).sum(), x, create_graph=True)
    second, = torch.autograd.grad(g.sum(), x)
    assert torch.equal(g, 3 * total.square()) and torch.allclose(second, 6 * total, rtol=1e-6)


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.filterwarnings("ignore")
def test_recording_is_refused(uf, call):
    """what would be recorded is the outputs' allocation: the replay would return the allocator's memory"""
    from torch.fx.experimental.proxy_tensor import make_fx
    o = operands()

    def run(x):
        return CALLS[call](uf, dict(o, x=x))

    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(run, o["x"], check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(run)(o["x"])
    leaf = o["x"].requires_grad_(True)
    out = run(leaf).sum()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(out, leaf, g, retain_graph=True)[0])(torch.ones_like(out))
    torch.autograd.grad(out, leaf)   # neither leaves anything behind


def test_modules_are_not_traced_either(uf):
    from geo_amd import utils_class
    layer = utils_class.Linear_Q8(24, 16).cuda().eval()
    layer.prepare()
    with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(layer, torch.ones(3, 24, device="cuda"), check_trace=False)
