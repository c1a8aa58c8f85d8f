"""Steps that go past the caches: the same bits as 32-bit operations one by one, and as the form that small or shifted tensors take."""
import ctypes

import pytest
import torch

from tests.test_gpu_adamw import ADAM_EPS, BETAS, DECAY, LR, eight, formula, uf, values  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def uncached(p, g, m, v, scales, copies, clamped):
    """whether the step of these tensors goes past the caches"""
    from geo_amd import _native
    place = lambda xs, i: xs[i].data_ptr() if xs else None   # noqa: E731
    tensors = (_native.AdamWTensor * len(p))(*[
        _native.AdamWTensor(param=p[i].data_ptr(), grad=g[i].data_ptr(), exp_avg=m[i].data_ptr(), exp_avg_sq=v[i].data_ptr(),
                            avg_scale=place(scales and scales[0], i), sq_scale=place(scales and scales[1], i), copy=place(copies, i),
                            clamped=place(clamped, i), elements=p[i].numel()) for i in range(len(p))])
    o = _native.AdamWOptions(struct_bytes=ctypes.sizeof(_native.AdamWOptions), state_bits=8 if scales else 32, lr=LR, beta1=BETAS[0], beta2=BETAS[1],
                             eps=ADAM_EPS, grad_scale=1.0, lo=-1, hi=1, step=1, param_dtype=TYPES[p[0].dtype], grad_dtype=TYPES[g[0].dtype],
                             copy_dtype=TYPES[copies[0].dtype] if copies else 0)
    launches, past = ctypes.c_int(), ctypes.c_int()
    assert _native.lib().geo_sc_adamw_plan(len(p), tensors, ctypes.byref(o), ctypes.byref(launches), ctypes.byref(past)) == 0
    return past.value


def normal(n, seed, scale, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)


def placed(xs, shift):
    """clones, each `shift` elements behind the start of an allocation"""
    out = []
    for x in xs:
        one = torch.empty(x.numel() + shift, dtype=x.dtype, device="cuda")[shift:]
        one.copy_(x)
        out.append(one)
    return out


# ragged counts: a chunk, a block and a workgroup cut; small tensors between large ones
@pytest.mark.parametrize("kinds", [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float32, torch.float32), (torch.float16, torch.float16, None)], ids=str)
def test_states_of_32_bits(uf, kinds):
    dtype, grad_type, copy_type = kinds
    sizes = [12_000_001, 7, 255, 3_000_003]
    p, g = [normal(n, 10 + i, 0.1, dtype) for i, n in enumerate(sizes)], [normal(n, 20 + i, 0.5, grad_type) for i, n in enumerate(sizes)]
    m, v = [normal(n, 30 + i, 0.01) for i, n in enumerate(sizes)], [normal(n, 40 + i, 0.02).square() for i, n in enumerate(sizes)]
    results = []
    for shift in (0, 1):
        lists = [placed(xs, shift) for xs in (p, g, m, v)]
        copies = [torch.zeros(n, dtype=copy_type, device="cuda") for n in sizes] if copy_type else None
        clamped = [torch.zeros(n, device="cuda") for n in sizes] if copy_type else None
        assert uncached(*lists, None, copies, clamped) == (shift == 0)
        uf.adamw_step(*lists, 7, LR, BETAS, ADAM_EPS, DECAY, 1 / 64, copies=copies, clamped=clamped, bounds=(-0.1, 0.05))
        results.append([lists[0], lists[2], lists[3]] + ([copies, clamped] if copies else []))
    for i in range(len(sizes)):
        want_p, want_m, want_v = formula(p[i], g[i], m[i], v[i], 7, 1 / 64, wide=False)
        for got in results:
            assert torch.equal(got[0][i], want_p.to(dtype)) and torch.equal(got[1][i], want_m) and torch.equal(got[2][i], want_v)
            if copy_type:
                assert torch.equal(got[3][i], want_p.to(copy_type)) and torch.equal(got[4][i], want_p.clamp(-0.1, 0.05))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_of_8_bits(uf, dtype):
    sizes = [40_000_001, 300, 1, 5_000_007]
    p, g = [normal(n, 10 + i, 0.1, dtype) for i, n in enumerate(sizes)], [normal(n, 20 + i, 0.5) for i, n in enumerate(sizes)]
    (m, ms), (r, rs) = (eight([normal(n, 30 + i, 0.01) for i, n in enumerate(sizes)]),
                        eight([normal(n, 40 + i, 0.02).abs() + 1e-3 for i, n in enumerate(sizes)]))
    results = []
    for shift in (0, 1):
        lists = [placed(xs, shift) for xs in (p, g, m, r, ms, rs)]
        assert uncached(*lists[:4], lists[4:], None, None) == (shift == 0)
        uf.adamw_step(*lists[:4], 5, LR, BETAS, ADAM_EPS, DECAY, scales=tuple(lists[4:]))
        results.append(lists)
    for i in range(len(sizes)):
        # the parameters do not see the rounding of the new states; those are the same codes in both forms
        want, want_m, _ = formula(p[i], g[i], values(m[i:i + 1], ms[i:i + 1])[0], values(r[i:i + 1], rs[i:i + 1])[0].square(), 5, wide=False)
        for got in results:
            assert torch.equal(got[0][i], want.to(dtype))
        for k in (2, 3, 4, 5):
            assert torch.equal(results[0][k][i].view(torch.uint8), results[1][k][i].view(torch.uint8)), k
        new = values(results[0][2][i:i + 1], results[0][4][i:i + 1])[0]
        unit = results[0][4][i].double().repeat_interleave(256)[:sizes[i]]
        step = torch.maximum(torch.exp2(torch.floor(torch.log2(want_m.double().abs().clamp(min=1e-30))) - 3), unit * 2.0 ** -9)
        assert ((new - want_m.double()).abs() < step * (1 + 1e-6)).all()
