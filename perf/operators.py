"""The 8-bit rows, the root-mean-square norm with 8-bit output, the 8-bit integer product and the distillation loss as
measured workloads: listed cases, a generator of further ones, their inputs, one pass through the operator (the framework's
kernels where ``own`` is true, elementary torch operations in 32 bits where it is not), the outputs in 64 bits, and what a
pass has to move and compute.

Operators (``op`` of a case) and what a pass returns:

``rows``     a scale per row and 8-bit integers of a matrix: the values that they stand for, the scales
``norm``     root-mean-square norm of ``x + residual`` with 8-bit output: the output's values, the sum;
             ``train``: also the gradients of x, the residual and the norm's weight
``product``  product of 8-bit matrices with a scale per row of either; ``train``: of the quantised rows of an activation
             and a weight, with the gradients of both
``distill``  divergence from a teacher's top logits, mean over the rows, with the gradient of the logits
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ------------------------------------------------------------------ cases

def listed():
    return [
        # output channels of a large weight brought to 8 bits when a checkpoint is loaded
        dict(name="rows_weight", op="rows", rows=16384, cols=4096, dtype="f32"),
        # a ragged batch of activations in front of an 8-bit product that no norm precedes
        dict(name="rows_ragged", op="rows", rows=1009, cols=1111, dtype="bf16"),
        # one token of a decoding loop: latency
        dict(name="norm_token", op="norm", rows=1, cols=4096, dtype="bf16", residual=True, train=False),
        # a training batch's tokens, not a round number of them
        dict(name="norm_train", op="norm", rows=8191, cols=4096, dtype="bf16", residual=True, train=True),
        # one token through a 4096 x 4096 layer: the weight is read once, latency counts
        dict(name="product_token", op="product", rows=1, cols=4096, inner=4096, dtype="bf16", train=False),
        # a decoding batch through the layer that narrows
        dict(name="product_batch", op="product", rows=48, cols=4096, inner=16384, dtype="bf16", train=False),
        # a long prompt through the layer that widens: the largest
        dict(name="product_prompt", op="product", rows=8192, cols=16384, inner=4096, dtype="bf16", train=False),
        # odd sizes everywhere, 32-bit tensors, forward and backward
        dict(name="product_ragged", op="product", rows=1009, cols=1003, inner=1111, dtype="f32", train=True),
        # a training step's layer, forward and backward
        dict(name="product_train", op="product", rows=4096, cols=4096, inner=4096, dtype="bf16", train=True),
        # a batch of images with ten classes
        dict(name="distill_classes", op="distill", rows=256, cols=10, top=5, dtype="f32", temperature=4.0),
        # a batch of tokens over a vocabulary
        dict(name="distill_words", op="distill", rows=4096, cols=32768, top=64, dtype="bf16", temperature=1.0),
        # few rows over a long odd vocabulary
        dict(name="distill_long", op="distill", rows=19, cols=100003, top=33, dtype="bf16", temperature=2.0),
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["rows", "norm", "norm", "product", "product", "product", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op in ("rows", "norm"):
        cols = size(16, 16384)
        case = dict(op=op, rows=size(1, min(16384, (1 << 25) // cols)), cols=cols, dtype=dtype)
        if op == "norm":
            case.update(residual=rng.random() < 0.7, train=rng.random() < 0.5)
        return case
    if op == "product":
        train = rng.random() < 0.4
        rows, cols, inner = size(1, 8192), size(16, 16384), size(16, 16384)
        most = (1 << 36) if train else (1 << 39)
        while rows * cols * inner > most:   # the largest side gives way
            if inner >= max(rows, cols):
                inner = inner * 2 // 3
            elif cols >= rows:
                cols = cols * 2 // 3
            else:
                rows = rows * 2 // 3
        return dict(op=op, rows=rows, cols=cols, inner=inner, dtype=dtype, train=train)
    cols = size(10, 131072)
    return dict(op=op, rows=size(1, min(4096, (1 << 27) // cols)), cols=cols, top=min(cols, size(1, 128)),
                dtype=dtype, temperature=rng.choice([1.0, 2.0, 4.0]))


# ------------------------------------------------------------------ inputs

def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device=gen.device) * scale


def _hidden(gen, rows, cols):
    """Hidden states: a few channels are much larger than the rest, rows differ in size."""
    wide = torch.where(torch.rand(cols, generator=gen, device=gen.device) < 0.01, 12.0, 1.0)
    return _normal(gen, rows, cols) * wide * torch.exp(_normal(gen, rows, 1, scale=0.3))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, rows, cols = TYPES[case["dtype"]], case["rows"], case["cols"]
    state = dict(case=case, dtype=dtype)
    if case["op"] == "rows":
        state["x"] = _hidden(gen, rows, cols).to(dtype)
    elif case["op"] == "norm":
        train = case["train"]
        state["x"] = _hidden(gen, rows, cols).to(dtype).requires_grad_(train)
        state["residual"] = _hidden(gen, rows, cols).to(dtype).requires_grad_(train) if case["residual"] else None
        state["weight"] = (1 + _normal(gen, cols, scale=0.1)).to(dtype).requires_grad_(train)
        if train:
            state["grad_values"] = _normal(gen, rows, cols, scale=1e-2).to(torch.bfloat16)   # the type of the values
            state["grad_total"] = _normal(gen, rows, cols, scale=1e-2).to(dtype) if case["residual"] else None
    elif case["op"] == "product":
        inner = case["inner"]
        x, w = _hidden(gen, rows, inner), _normal(gen, cols, inner, scale=inner ** -0.5)
        if case["train"]:
            state["x"], state["w"] = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
            state["grad"] = _normal(gen, rows, cols, scale=1e-2).to(dtype)
        else:   # a serving program holds its weights in 8 bits; the activations come so from the norm before
            state["q"], state["scale"] = _rows(x)
            state["wq"], state["wscale"] = _rows(w)
            for k in ("q", "wq"):
                state[k] = state[k].to(torch.int8)
            for k in ("scale", "wscale"):
                state[k] = state[k].reshape(-1)
    else:
        shared = _normal(gen, rows, cols, scale=2.0)
        top = (shared + _normal(gen, rows, cols, scale=0.7)).topk(case["top"], dim=1)
        state["z"] = (shared + _normal(gen, rows, cols)).to(dtype).requires_grad_(True)
        state["top_logits"], state["top_index"] = top.values.to(dtype), top.indices.to(torch.int32)
        if rows > 16:   # a padded position has no entries, another one fewer than the others
            state["top_index"][rows // 3] = -1
            state["top_index"][rows // 2, case["top"] // 2:] = -1
        state["grad"] = torch.tensor(128.0, device="cuda")   # the training loop's loss scale
    return state


# ------------------------------------------------------------------ plain form: elementary operations in 32 bits

def _rows(n):
    most = n.abs().amax(-1, keepdim=True)
    q = (n * torch.where(most > 0, torch.full_like(most, 127.0) / most, 0.0)).round()
    return q, most * (1.0 / 127.0)


def _plain_rows(state):
    q, scale = _rows(state["x"].float())
    return dict(values=(q * scale).to(torch.bfloat16), scale=scale.reshape(-1))


def _plain_norm(state):
    dtype, weight = state["dtype"], state["weight"].detach().float()
    total = state["x"].detach().float()
    if state["residual"] is not None:
        total = total + state["residual"].detach().float()
    rstd = 1.0 / torch.sqrt(total.square().mean(-1, keepdim=True) + EPS)
    q, scale = _rows(total * rstd * weight)
    out = dict(values=(q * scale).to(torch.bfloat16), total=total.to(dtype))
    if state["case"]["train"]:
        grad = state["grad_values"].float()
        u = grad * weight
        dx = rstd * (u - total * rstd.square() * (u * total).mean(-1, keepdim=True))
        if state["grad_total"] is not None:
            dx = dx + state["grad_total"].float()
        dx = dx.to(dtype)
        out.update(dx=dx, dweight=(grad * total * rstd).sum(0).to(dtype))
        if state["residual"] is not None:
            out["dresidual"] = dx
    return out


def _plain_product(state):
    dtype = state["dtype"]
    if not state["case"]["train"]:
        y = (state["q"].float() @ state["wq"].float().t()) * state["scale"][:, None] * state["wscale"]
        return dict(y=y.to(dtype))
    (q, scale), (wq, wscale) = _rows(state["x"].detach().float()), _rows(state["w"].detach().float())
    x, w, grad = q * scale, wq * wscale, state["grad"].float()
    return dict(y=(x @ w.t()).to(dtype), dx=(grad @ w).to(dtype), dw=(grad.t() @ x).to(dtype))


def _plain_distill(state):
    temperature, z = state["case"]["temperature"], state["z"].detach().float() / state["case"]["temperature"]
    index = state["top_index"].long()
    there = index >= 0
    t = torch.where(there, state["top_logits"].float() / temperature, -torch.inf)
    some = there.any(1, keepdim=True)
    t = t - torch.where(some, t.amax(1, keepdim=True), 0.0)
    p = t.exp()
    total = torch.where(some, p.sum(1, keepdim=True), 1.0)
    p, log_p = p / total, t - total.log()
    shifted = z - z.amax(1, keepdim=True)
    e = shifted.exp()
    norm = e.sum(1, keepdim=True)
    log_q = shifted.gather(1, index.clamp(min=0)) - norm.log()
    loss = torch.where(there, p * (log_p - log_q), 0.0).sum() * (temperature ** 2 / z.shape[0])
    dz = (e / norm * some).scatter_add(1, index.clamp(min=0), -p) * (state["grad"] * (temperature / z.shape[0]))
    return dict(loss=loss, dz=dz.to(state["dtype"]))


# ------------------------------------------------------------------ the framework's kernels

def _own_rows(state):
    from geo_amd import utils_functional as uf
    _, scale, values = uf.quantize_rows(state["x"], values=torch.bfloat16)
    return dict(values=values, scale=scale)


def _own_norm(state):
    from geo_amd import utils_functional as uf
    x, residual, weight = state["x"], state["residual"], state["weight"]
    _, _, total, values = uf.rms_norm_q8(x, weight, residual=residual, eps=EPS, values=torch.bfloat16)
    out = dict(values=values, total=total)
    if state["case"]["train"]:
        grad = state["grad_values"]
        if residual is not None:
            out["dx"], out["dresidual"], out["dweight"] = torch.autograd.grad(
                (values, total), (x, residual, weight), (grad, state["grad_total"]))
        else:
            out["dx"], out["dweight"] = torch.autograd.grad((values,), (x, weight), (grad,))
    return out


def _own_product(state):
    from geo_amd import utils_functional as uf
    if not state["case"]["train"]:
        return dict(y=uf.matmul_q8(state["q"], state["scale"], state["wq"], state["wscale"], dtype=state["dtype"]))
    y = uf.linear_q8(state["x"], state["w"])
    dx, dw = torch.autograd.grad((y,), (state["x"], state["w"]), (state["grad"],))
    return dict(y=y, dx=dx, dw=dw)


def _own_distill(state):
    from geo_amd import utils_functional as uf
    loss = uf.distill_topk(state["z"], state["top_logits"], state["top_index"],
                           temperature=state["case"]["temperature"])
    dz, = torch.autograd.grad((loss,), (state["z"],), (state["grad"],))
    return dict(loss=loss, dz=dz)


PLAIN = dict(rows=_plain_rows, norm=_plain_norm, product=_plain_product, distill=_plain_distill)
OWN = dict(rows=_own_rows, norm=_own_norm, product=_own_product, distill=_own_distill)


def run(state):
    op = state["case"]["op"]
    if own:
        return OWN[op](state)
    with torch.no_grad():
        return PLAIN[op](state)


# ------------------------------------------------------------------ outputs in 64 bits

def _eighth(v):
    """The values that rows of 64-bit numbers have in 8 bits, and their scales."""
    largest = v.abs().max(dim=1).values
    step = largest / 127
    safe = torch.where(step > 0, step, torch.ones_like(step))
    return torch.round(v / safe[:, None]) * step[:, None], step


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["op"] == "rows":
        values, step = _eighth(wide["x"])
        return dict(values=values, scale=step)
    if case["op"] == "norm":
        total = wide["x"] + wide.get("residual", 0.0)
        inverse = (torch.einsum("rc,rc->r", total, total) / case["cols"] + EPS).rsqrt()[:, None]
        unit = total * inverse
        out = dict(values=_eighth(unit * wide["weight"])[0], total=total)
        if case["train"]:
            g = wide["grad_values"] * wide["weight"]
            along = torch.einsum("rc,rc->r", g, unit)[:, None] / case["cols"]
            out["dx"] = (g - unit * along) * inverse + wide.get("grad_total", 0.0)
            out["dweight"] = torch.einsum("rc,rc->c", wide["grad_values"], unit)
            if case["residual"]:
                out["dresidual"] = out["dx"]
        return out
    if case["op"] == "product":
        if not case["train"]:
            a = state["q"].double() * wide["scale"][:, None]
            return dict(y=torch.mm(a, (state["wq"].double() * wide["wscale"][:, None]).t()))
        a, b = _eighth(wide["x"])[0], _eighth(wide["w"])[0]
        return dict(y=torch.mm(a, b.t()), dx=torch.mm(wide["grad"], b), dw=torch.mm(wide["grad"].t(), a))
    temperature, index = case["temperature"], state["top_index"].long()
    log_q = torch.log_softmax(wide["z"] / temperature, dim=1)
    teacher = torch.zeros_like(log_q)
    loss = torch.zeros((), dtype=torch.float64, device=log_q.device)
    for r in range(case["rows"]):
        at = index[r][index[r] >= 0]
        if at.numel():
            log_p = torch.log_softmax(wide["top_logits"][r][index[r] >= 0] / temperature, dim=0)
            teacher[r, at] = log_p.exp()
            loss += (log_p.exp() * (log_p - log_q[r, at])).sum()
        else:
            log_q[r] = -torch.inf   # no gradient
    scale = temperature ** 2 / case["rows"]
    return dict(loss=loss * scale, dz=(log_q.exp() - teacher) * (wide["grad"] * scale / temperature))


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    rows, cols, size = case["rows"], case["cols"], TYPES[case["dtype"]].itemsize
    cells = rows * cols
    if case["op"] == "rows":
        return dict(bytes=cells * (size + 2) + 4 * rows, flops=4 * cells)
    if case["op"] == "norm":
        moved = size + 2 + (2 * size if case["residual"] else 0)       # x, values; residual, sum
        if case["train"]:
            moved += 2 + size + (size if case["residual"] else 0)      # gradient of the values, dx; gradient of the sum
        return dict(bytes=cells * moved + cols * size, flops=cells * (20 if case["train"] else 8))
    if case["op"] == "product":
        inner = case["inner"]
        if not case["train"]:
            return dict(bytes=(rows + cols) * (inner + 4) + cells * size, flops=2 * cells * inner)
        # x, w, the gradient in; y, dx, dw out
        return dict(bytes=2 * size * (rows * inner + cols * inner + cells), flops=6 * cells * inner)
    return dict(bytes=2 * size * cells + rows * case["top"] * (size + 4), flops=8 * cells)
