"""The tensors of a step that belong together have one shape: as many elements in another order would be other elements."""
import pytest
import torch

from tests.test_gpu_adamw import uf  # noqa: F401

pytestmark = pytest.mark.gpu


def test_refused(uf):
    x = lambda *s: torch.zeros(*s, device="cuda")   # noqa: E731
    p, g, m, v = [x(2, 3)], [torch.ones(2, 3, device="cuda")], [x(2, 3)], [x(2, 3)]
    for lists in ((p, [x(3, 2)], m, v), (p, [x(6)], m, v), (p, [x(1, 2, 3)], m, v), (p, g, [x(3, 2)], v), (p, g, m, [x(6)])):
        with pytest.raises(RuntimeError, match="shape"):
            uf.adamw_step(*lists, 1, 0.1)
    for more in (dict(copies=[x(3, 2)]), dict(clamped=[x(6)])):
        with pytest.raises(RuntimeError, match="shape"):
            uf.adamw_step(p, g, m, v, 1, 0.1, **more)
    eight = [[x(3, 2).to(torch.float8_e4m3fn)], [x(2, 3).to(torch.float8_e4m3fn)]]
    with pytest.raises(RuntimeError, match="shape"):
        uf.adamw_step(p, g, *eight, 1, 0.1, scales=tuple([torch.zeros(1, device="cuda", dtype=torch.float8_e8m0fnu)] for _ in range(2)))
    assert (p[0] == 0).all() and (m[0] == 0).all()
    uf.adamw_step(p, g, m, v, 1, 0.1, weight_decay=0.0, copies=[x(2, 3)], clamped=[x(2, 3)])
    assert (p[0] + 0.1).abs().max() < 1e-6


def test_saved_states_of_another_shape(uf):
    from geo_amd import network
    p = torch.ones(2, 3, device="cuda", requires_grad=True)
    p.grad = torch.ones(2, 3, device="cuda")
    opt = network.AdamW([p])
    opt.step()
    saved = opt.state_dict()
    saved["state"][0]["exp_avg"] = saved["state"][0]["exp_avg"].reshape(3, 2)
    with pytest.raises(ValueError, match="does not fit"):
        network.AdamW([p]).load_state_dict(saved)
