"""A layer's prepared weight: what keeps it, what drops it, and that an outdated one does not serve unnoticed."""
import copy
import io
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["Linear_Q8", "NormLinear_Q8"])
def layer(request):
    from geo_amd import utils_class
    torch.manual_seed(0)
    return getattr(utils_class, request.param)(48, 20).cuda()


@pytest.fixture(autouse=True)
def no_gradients():
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("error")
        yield


def value(layer, x):
    y = layer(x)
    return y[0] if isinstance(y, tuple) else y


X = torch.randn(7, 48, generator=torch.Generator().manual_seed(1))


def test_eval_keeps_it_and_train_drops_it(layer):
    x = X.cuda()
    want = value(layer, x)
    layer.prepare()
    layer.eval()
    assert layer._q8 is not None and torch.equal(value(layer, x), want)
    layer.train()
    assert layer._q8 is None and torch.equal(value(layer, x), want)


def test_another_type_or_device_drops_it(layer):
    x = X.cuda().bfloat16()
    layer.eval().prepare()
    layer.cuda()                                 # where it is already: nothing changes
    assert layer._q8 is not None
    other = copy.deepcopy(layer).bfloat16()
    assert other._q8 is None
    plain = copy.deepcopy(layer).train()
    assert torch.equal(value(other, x), value(copy.deepcopy(plain).bfloat16(), x))
    layer.cpu()
    assert layer._q8 is None
    layer.cuda()
    assert torch.equal(value(layer, X.cuda()), value(plain, X.cuda()))


def test_an_outdated_one_is_warned_of(layer):
    x = X.cuda()
    layer.eval().prepare()
    old = value(layer, x)
    layer.weight.mul_(torch.linspace(1, 2, 20, device="cuda")[:, None])
    with pytest.warns(UserWarning, match="prepare"):
        assert torch.equal(value(layer, x), old)
    with torch.enable_grad():                    # gradients are the weight's own
        new = value(layer, x).detach()
    assert not torch.equal(new, old)
    layer.prepare()
    assert torch.equal(value(layer, x), new)
    layer.weight.data = layer.weight.data.clone()   # re-pointed, as train_step does with masters
    with pytest.warns(UserWarning, match="prepare"):
        value(layer, x)


def test_copies_are_prepared_as_their_original_is(layer):
    x = X.cuda()
    layer.eval().prepare()
    want = value(layer, x)
    buffer = io.BytesIO()
    torch.save(layer, buffer)
    buffer.seek(0)
    for other in (copy.deepcopy(layer), torch.load(buffer, weights_only=False)):
        assert other._q8 is not None and torch.equal(value(other, x), want)
    layer.weight.mul_(-1)
    other = copy.deepcopy(layer)
    assert other._q8 is None and torch.equal(value(other, x), -want)


def test_in_inference_mode():
    from geo_amd import utils_class
    with torch.inference_mode():
        layer = utils_class.NormLinear_Q8(48, 20).cuda().eval()
        want = value(layer, X.cuda())
        layer.prepare()
        assert torch.equal(value(layer, X.cuda()), want)
