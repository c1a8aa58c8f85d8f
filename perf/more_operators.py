"""The 8-bit product with bias, activation and residual in its epilogue, the gated norm between two blocks and the AdamW step over many
tensors as measured workloads: listed cases, a generator of further ones, their inputs, one pass through the operator (the
framework's kernels where ``own`` is true, elementary torch operations where it is not), the outputs in 64 bits, and what a
pass has to move and compute.

Operators (``op`` of a case) and what a pass returns:

``product``  act(x w^T + bias) + residual of 8-bit rows with a scale each; ``train``: of the quantised rows of an activation and a
             weight, with the gradients of all four
``norm``     total = residual_scale residual + gate norm(x) post_weight, and norm(total) weight; ``train``: with the gradients of all
             six; ``eight``: the second norm's output in 8 bits, returned as the values it stands for
``adamw``    one AdamW step on a list of tensors that lie in flat buffers: the parameters, both moments (states of 8 bits: the
             codes as float8 numbers, and their scales, powers of two), and the copies that the step writes

A relu in training has 16-bit types only: in 32 bits a single number on the other side of zero changes a gradient by more than all
roundings together.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
LR, BETAS, ADAM_EPS, DECAY, LOSS_SCALE = 1e-3, (0.9, 0.999), 1e-8, 0.01, 128.0
FIRST_STEP = 100        # a run in progress
BLOCK = 256             # elements of a tensor that share a scale of 8-bit states
BOUNDS = (-1.0, 0.999)  # of the clamped copies

# elements of the parameters of network.CONV_tiny_add_partial and network.PatchMLP_q8
NETWORKS = {
    "cnn": [32, 32, 32, 32, 64, 64, 10, 10, 32 * 3 * 25, 32 * 32 * 25, 64 * 32 * 25, 10 * 64 * 16],
    "teacher": [256 * 48] + [1024 * 256, 256] * 4 + [256 * 1024] * 4 + [10 * 256, 256],
}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one token through the layer that widens: latency, the weight is read once
        dict(name="product_token", op="product", rows=1, cols=16384, inner=4096, dtype="bf16", activation="gelu", bias=True,
             residual=False, train=False),
        # a long prompt through the layer that narrows, onto the residual stream: the largest
        dict(name="product_prompt", op="product", rows=8192, cols=4096, inner=16384, dtype="bf16", activation="none", bias=True,
             residual=True, train=False),
        # PatchMLP_q8's widening layer in training: 256 images of 64 patches, short inner dimension
        dict(name="product_images", op="product", rows=16384, cols=1024, inner=256, dtype="bf16", activation="relu", bias=True,
             residual=False, train=True),
        # a training step's layer with all there is, odd sizes everywhere
        dict(name="product_train", op="product", rows=4095, cols=4099, inner=2047, dtype="bf16", activation="silu", bias=True,
             residual=True, train=True),
        # one token of a served network, in front of an 8-bit product: latency
        dict(name="norm_token", op="norm", rows=1, cols=4096, dtype="bf16", post=True, gate=1, scale=True, train=False, eight=True),
        # PatchMLP_q8's rows of a batch in training, a gate per channel
        dict(name="norm_images", op="norm", rows=16384, cols=256, dtype="f32", post=True, gate=1, scale=False, train=True, eight=False),
        # a training batch of 16 samples with a gate each
        dict(name="norm_train", op="norm", rows=8192, cols=4096, dtype="bf16", post=True, gate=16, scale=True, train=True, eight=False),
        # odd sizes, no norm behind the block, no gate
        dict(name="norm_ragged", op="norm", rows=1009, cols=1111, dtype="f16", post=False, gate=0, scale=True, train=True, eight=False),
        # the 4-layer SC network's step: masters, scaled gradients, copies into parameters and clamped buffers; latency
        dict(name="adamw_cnn", op="adamw", network="cnn", bits=32, dtype="f32", grad="f32", copy="f32", clamp=True),
        # the teacher's step with 8-bit states
        dict(name="adamw_teacher", op="adamw", network="teacher", bits=8, dtype="f32", grad="f32", copy="none", clamp=False),
        # masters of a large network with 16-bit gradients and parameters
        dict(name="adamw_masters", op="adamw", network="", tensors=96, largest=1 << 24, ratio=0.88, bits=32, dtype="f32", grad="bf16",
             copy="bf16", clamp=False),
        # the same in 8-bit states, odd sizes
        dict(name="adamw_eight", op="adamw", network="", tensors=61, largest=16777213, ratio=0.86, bits=8, dtype="f32", grad="bf16",
             copy="bf16", clamp=False),
    ]


def draw(rng):
    def size(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["product", "product", "product", "norm", "norm", "norm", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op == "product":
        train = rng.random() < 0.5
        rows, cols, inner = size(1, 16384), size(16, 16384), size(16, 16384)
        most = (1 << 36) if train else (1 << 39)
        while rows * cols * inner > most:   # the largest side gives way
            if inner >= max(rows, cols):
                inner = inner * 2 // 3
            elif cols >= rows:
                cols = cols * 2 // 3
            else:
                rows = rows * 2 // 3
        kinds = ["none", "gelu", "silu"] + (["relu"] if dtype != "f32" or not train else [])
        return dict(op=op, rows=rows, cols=cols, inner=inner, dtype=dtype, activation=rng.choice(kinds),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train)
    if op == "norm":
        cols = size(16, 16384)
        rows = size(1, min(16384, (1 << 25) // cols))
        runs = rng.choice([0, 1, 1, 2, 3, 16, rows])
        train = rng.random() < 0.6
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, post=rng.random() < 0.7, gate=runs if runs and rows % runs == 0 else 1,
                    scale=rng.random() < 0.5, train=train, eight=not train and rng.random() < 0.5)
    largest, ratio = size(100, 1 << 23), rng.choice([0.6, 0.8, 0.9, 1.0])
    return dict(op=op, network="", tensors=size(1, 200 if largest < 1 << 20 else 16), largest=largest, ratio=ratio, bits=rng.choice([8, 32]),
                dtype=dtype, grad=rng.choice([dtype, "f32"]), copy=rng.choice(["none", "f32", "bf16", "f16"]), clamp=rng.random() < 0.3)


def _sizes(case):
    """Elements of the tensors of an AdamW case."""
    if case["network"]:
        return NETWORKS[case["network"]]
    return [max(1, int(case["largest"] * case["ratio"] ** i)) for i in range(case["tensors"])]


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
    state = dict(case=case, dtype=TYPES[case["dtype"]])
    dict(product=_prepare_product, norm=_prepare_norm, adamw=_prepare_adamw)[case["op"]](case, gen, state)
    return state


def _prepare_product(case, gen, state):
    dtype, rows, cols, inner, train = state["dtype"], case["rows"], case["cols"], case["inner"], case["train"]
    x, w = _hidden(gen, rows, inner), _normal(gen, cols, inner, scale=inner ** -0.5)
    state["bias"] = _normal(gen, cols, scale=0.3).to(dtype).requires_grad_(train) if case["bias"] else None
    state["residual"] = _hidden(gen, rows, cols).to(dtype).requires_grad_(train) if case["residual"] else None
    if train:
        state["x"], state["w"] = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
        state["grad"] = _normal(gen, rows, cols, scale=1e-2).to(dtype)
    else:   # a serving program holds its weights in 8 bits; the activations come so from the norm before
        for q, scale, v in (("q", "scale", x), ("wq", "wscale", w)):
            state[q], state[scale] = _rows(v)
            state[q], state[scale] = state[q].to(torch.int8), state[scale].reshape(-1)


def _prepare_norm(case, gen, state):
    dtype, rows, cols, train = state["dtype"], case["rows"], case["cols"], case["train"]
    state["x"] = (_hidden(gen, rows, cols) * 0.5).to(dtype).requires_grad_(train)
    state["residual"] = _hidden(gen, rows, cols).to(dtype).requires_grad_(train)
    around_one = lambda *shape: (1 + _normal(gen, *shape, scale=0.1)).to(dtype).requires_grad_(train)   # noqa: E731
    state["weight"] = around_one(cols)
    state["post"] = around_one(cols) if case["post"] else None
    state["scale"] = around_one(cols) if case["scale"] else None
    state["gate"] = None
    if case["gate"]:   # of every channel, or of every run of rows (a sample's tokens)
        runs = case["gate"]
        state["gate"] = _normal(gen, runs, cols, scale=0.5).to(dtype)
        state["gate"] = (state["gate"].reshape(cols) if runs == 1 else state["gate"]).requires_grad_(train)
    if train:
        state["grad_out"] = _normal(gen, rows, cols, scale=1e-2).to(dtype)
        state["grad_total"] = _normal(gen, rows, cols, scale=1e-2).to(dtype)


def _prepare_adamw(case, gen, state):
    """Tensors as views of flat buffers, each at a multiple of BLOCK elements; what lies between them is zero and stays so."""
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    there = torch.zeros(total, dtype=torch.bool, device="cuda")
    parts = list(zip(starts, sizes))
    for at, n in parts:
        there[at:at + n] = True
    # magnitudes differ from block to block, as they do from channel to channel
    level = torch.exp(_normal(gen, total // BLOCK, scale=1.0)).repeat_interleave(BLOCK)
    draw_one = lambda scale: torch.where(there, _normal(gen, total, scale=scale), 0.0)   # noqa: E731
    flat = dict(p=draw_one(0.05).to(state["dtype"]), g=(draw_one(1e-3 * LOSS_SCALE) * level).to(TYPES[case["grad"]]))
    m = draw_one(3e-4) * level
    root = torch.where(there, draw_one(1e-3).abs() * level * 0.3 + 7e-4 * level, 0.0)
    if case["bits"] == 8:
        for name, v in (("m", m), ("v", root)):
            scale = _block_scale(v.reshape(-1, BLOCK))
            flat[name] = (v.reshape(-1, BLOCK) / scale).to(torch.float8_e4m3fn).reshape(-1)
            flat[name + "_scale"] = scale.reshape(-1).to(torch.float8_e8m0fnu)
    else:
        flat.update(m=m, v=root.square())
    if case["copy"] != "none":
        flat["copy"] = torch.zeros(total, dtype=TYPES[case["copy"]], device="cuda")
    if case["clamp"]:
        flat["clamped"] = torch.zeros(total, dtype=torch.float32, device="cuda")
    scales = [k for k in flat if k.endswith("_scale")]
    state["lists"] = {k: [v[at // BLOCK:(at + n - 1) // BLOCK + 1] if k in scales else v[at:at + n] for at, n in parts]
                      for k, v in flat.items()}
    state.update(flat=flat, step=FIRST_STEP)


# ------------------------------------------------------------------ plain form: elementary operations in 32 bits

def _rows(n):
    most = n.abs().amax(-1, keepdim=True)
    q = (n * torch.where(most > 0, torch.full_like(most, 127.0) / most, 0.0)).round()
    return q, most * (1.0 / 127.0)


def _activate(z, kind):
    """The activation and its slope."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if kind == "gelu":
        below = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * below, below + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def _plain_product(state):
    dtype, case = state["dtype"], state["case"]
    if case["train"]:
        (q, scale), (wq, wscale) = _rows(state["x"].detach().float()), _rows(state["w"].detach().float())
    else:
        q, scale, wq, wscale = state["q"].float(), state["scale"][:, None], state["wq"].float(), state["wscale"][:, None]
    z = (q @ wq.t()) * scale * wscale.t()
    if state["bias"] is not None:
        z = z + state["bias"].detach().float()
    y, slope = _activate(z, case["activation"])
    if state["residual"] is not None:
        y = y + state["residual"].detach().float()
    out = dict(y=y.to(dtype))
    if case["train"]:
        dz = state["grad"].float() * slope
        out.update(dx=(dz @ (wq * wscale)).to(dtype), dw=(dz.t() @ (q * scale)).to(dtype))
        if state["bias"] is not None:
            out["dbias"] = dz.sum(0).to(dtype)
        if state["residual"] is not None:
            out["dresidual"] = state["grad"]
    return out


def _unit(t):
    """A row over its root mean square, and that factor."""
    r = 1.0 / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)
    return t * r, r


def _plain_norm(state):
    dtype, case = state["dtype"], state["case"]
    x, residual, weight = (state[k].detach().float() for k in ("x", "residual", "weight"))
    post, gate, scale = (state[k].detach().float() if state[k] is not None else None for k in ("post", "gate", "scale"))
    runs = max(case["gate"], 1)
    spread = (lambda v: v.reshape(runs, 1, -1).expand(runs, case["rows"] // runs, -1).reshape(x.shape))
    n1, r1 = _unit(x) if post is not None else (x, None)
    m = n1 * post if post is not None else n1
    every_gate = spread(gate) if gate is not None else None
    gated = m * every_gate if gate is not None else m
    total = (residual * scale if scale is not None else residual) + gated
    n2, r2 = _unit(total)
    out = dict(total=total.to(dtype))
    if case["eight"]:
        q, step = _rows(n2 * weight)
        out["values"] = (q * step).to(torch.bfloat16)
        return out
    out["out"] = (n2 * weight).to(dtype)
    if case["train"]:
        grad = state["grad_out"].float()
        u = grad * weight
        dt = r2 * (u - n2 * (u * n2).mean(-1, keepdim=True)) + state["grad_total"].float()
        out["dweight"] = (grad * n2).sum(0).to(dtype)
        out["dresidual"] = (dt * scale if scale is not None else dt).to(dtype)
        if scale is not None:
            out["dscale"] = (dt * residual).sum(0).to(dtype)
        if gate is not None:
            out["dgate"] = (dt * m).reshape(runs, -1, case["cols"]).sum(1).reshape(gate.shape).to(dtype)
            dt = dt * every_gate
        if post is not None:
            out["dpost"] = (dt * n1).sum(0).to(dtype)
            dt = dt * post
            dt = r1 * (dt - n1 * (dt * n1).mean(-1, keepdim=True))
        out["dx"] = dt.to(dtype)
    return out


def _block_scale(v):
    """The power of two for each row of v that brings its largest number to 128 .. 256 (float8_e4m3fn ends at 448)."""
    field = (v.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 7
    return (field.clamp(min=1) << 23).view(torch.float32)


def _to_eight(v, dither):
    """v in float8_e4m3fn, up or down by `dither`, whole numbers of 32 bits that stand for a fraction of a step."""
    tiny = v < 2.0 ** -6   # below it the steps are 2^-9 throughout
    lifted = torch.where(tiny, v + 2.0 ** -6, v).view(torch.int32)
    kept = ((lifted + (dither >> 12).to(torch.int32)) & ~0xfffff).view(torch.float32)
    return torch.where(tiny, kept - 2.0 ** -6, kept)


def _dither(step, device):
    """For the places of a block: two sequences that fill [0, 2^32) evenly over places and over steps."""
    place = torch.arange(BLOCK, dtype=torch.int64, device=device)
    first = (place * 0x9E3779B1 + step * 0x6A09E667) & 0xffffffff
    return first, (first + 0x80000000) & 0xffffffff


def _plain_adamw(state):
    flat, case = state["flat"], state["case"]
    state["step"] += 1
    eight, step, (b1, b2) = case["bits"] == 8, state["step"], BETAS
    g = flat["g"].float() * (1.0 / LOSS_SCALE)
    if eight:
        m = (flat["m"].float().reshape(-1, BLOCK) * flat["m_scale"].float()[:, None]).reshape(-1)
        root = (flat["v"].float().reshape(-1, BLOCK) * flat["v_scale"].float()[:, None]).reshape(-1)
        v = root * root
    else:
        m, v = flat["m"], flat["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    p = flat["p"].float() * (1 - LR * DECAY)
    p = p - (m * (LR / (1 - b1 ** step))) / (root * (1 / math.sqrt(1 - b2 ** step)) + ADAM_EPS)
    flat["p"].copy_(p)
    if eight:
        for name, value, dither in zip("mv", (m, root), _dither(step, p.device)):
            rows = value.reshape(-1, BLOCK)
            scale = _block_scale(rows)
            codes = _to_eight((rows / scale).abs(), dither)
            if name == "v":
                codes = torch.where(rows > 0, codes.clamp(min=2.0 ** -9), 0.0)
            flat[name].copy_((codes * torch.where(rows < 0, -1.0, 1.0)).reshape(-1).to(torch.float8_e4m3fn))
            flat[name + "_scale"].copy_(scale.reshape(-1).to(torch.float8_e8m0fnu))
    else:
        flat["m"].copy_(m)
        flat["v"].copy_(v)
    if "copy" in flat:
        flat["copy"].copy_(p)
    if "clamped" in flat:
        flat["clamped"].copy_(p.clamp(*BOUNDS))
    return {k: v for k, v in flat.items() if k != "g"}


# ------------------------------------------------------------------ the framework's kernels

def _own_product(state):
    from geo_amd import utils_functional as uf
    case = state["case"]
    epilogue = dict(bias=state["bias"], activation=None if case["activation"] == "none" else case["activation"], residual=state["residual"])
    if not case["train"]:
        return dict(y=uf.matmul_q8(state["q"], state["scale"], state["wq"], state["wscale"], dtype=state["dtype"], **epilogue))
    y = uf.linear_q8(state["x"], state["w"], **epilogue)
    names = ["x", "w"] + [k for k in ("bias", "residual") if state[k] is not None]
    grads = torch.autograd.grad((y,), [state[k] for k in names], (state["grad"],))
    return dict(y=y, **{"d" + k: g for k, g in zip(names, grads)})


def _own_norm(state):
    from geo_amd import utils_functional as uf
    case = state["case"]
    gate = state["gate"]
    x, residual = state["x"], state["residual"]
    if case["gate"] > 1:   # (samples, rows of a sample, columns), the gate (samples, 1, columns)
        x, residual, gate = x.unflatten(0, (case["gate"], -1)), residual.unflatten(0, (case["gate"], -1)), gate.unsqueeze(1)
    around = dict(post_weight=state["post"], gate=gate, residual_scale=state["scale"], eps=EPS)
    if case["eight"]:
        _, _, total, values = uf.gated_norm_q8(x, residual, state["weight"], values=torch.bfloat16, **around)
        return dict(total=total.reshape(state["x"].shape), values=values.reshape(state["x"].shape))
    out, total = uf.gated_norm(x, residual, state["weight"], **around)
    result = dict(out=out.reshape(state["x"].shape), total=total.reshape(state["x"].shape))
    if case["train"]:
        names = ["x", "residual", "weight"] + [k for k in ("post", "gate", "scale") if state[k] is not None]
        grads = torch.autograd.grad((out, total), [state[k] for k in names],
                                    (state["grad_out"].reshape(out.shape), state["grad_total"].reshape(out.shape)))
        result.update({"d" + k: g for k, g in zip(names, grads)})
    return result


def _own_adamw(state):
    from geo_amd import utils_functional as uf
    lists = state["lists"]
    state["step"] += 1
    scales = (lists["m_scale"], lists["v_scale"]) if state["case"]["bits"] == 8 else None
    uf.adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], state["step"], lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
                  grad_scale=1.0 / LOSS_SCALE, scales=scales, copies=lists.get("copy"), clamped=lists.get("clamped"), bounds=BOUNDS)
    return {k: v for k, v in state["flat"].items() if k != "g"}


PLAIN = dict(product=_plain_product, norm=_plain_norm, adamw=_plain_adamw)
OWN = dict(product=_own_product, norm=_own_norm, adamw=_own_adamw)


def run(state):
    op = state["case"]["op"]
    if own:
        return OWN[op](state)
    with torch.no_grad():
        return PLAIN[op](state)


# ------------------------------------------------------------------ outputs in 64 bits

def _eighth(v):
    """The values that rows of 64-bit numbers have in 8 bits."""
    largest = v.abs().max(dim=1).values
    step = largest / 127
    safe = torch.where(step > 0, step, torch.ones_like(step))
    return torch.round(v / safe[:, None]) * step[:, None]


def _in_rows(v):
    """The values that rows have in 8 bits as the operator defines them: whole numbers from 32-bit operations, a step of 64 bits."""
    largest = v.float().abs().max(dim=1, keepdim=True).values
    inverse = torch.reciprocal(largest.double()).mul(127).nan_to_num(posinf=0.0).float()
    return torch.round(v.float() * inverse).double() * largest.double().div(127)


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.is_floating_point()}
    return dict(product=_exact_product, norm=_exact_norm, adamw=_exact_adamw)[case["op"]](case, state, wide)


def _exact_product(case, state, wide):
    if case["train"]:
        a, b = (_in_rows(state[k].detach()) for k in ("x", "w"))
    else:
        a, b = state["q"].double() * wide["scale"][:, None], state["wq"].double() * wide["wscale"][:, None]
    z = torch.mm(a, b.t())
    if case["bias"]:
        z += wide["bias"]
    kind = case["activation"]
    if kind == "gelu":
        y = torch.special.erfc(z / -math.sqrt(2)) / 2 * z
    elif kind == "silu":
        y = torch.sigmoid(z) * z
    else:
        y = torch.relu(z) if kind == "relu" else z.clone()
    if case["residual"]:
        y += wide["residual"]
    out = dict(y=y)
    if case["train"]:
        if kind == "gelu":
            slope = torch.special.erfc(z / -math.sqrt(2)) / 2 + z * torch.exp(z.square() / -2) / math.sqrt(2 * math.pi)
        elif kind == "silu":
            slope = torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
        else:
            slope = torch.heaviside(z, torch.zeros_like(z)) if kind == "relu" else torch.ones_like(z)
        dz = wide["grad"] * slope
        out.update(dx=torch.mm(dz, b), dw=torch.mm(dz.t(), a))
        if case["bias"]:
            out["dbias"] = torch.einsum("rc->c", dz)
        if case["residual"]:
            out["dresidual"] = wide["grad"]
    return out


def _exact_norm(case, state, wide):
    """The forward written out; the gradients by 64-bit autograd of it."""
    runs = max(case["gate"], 1)
    leaves = {k: v.requires_grad_(True) for k, v in wide.items() if not k.startswith("grad")}
    branch = leaves["x"]
    if case["post"]:
        branch = branch / torch.linalg.vector_norm(torch.cat([branch, torch.full_like(branch[:, :1], math.sqrt(EPS * case["cols"]))], 1),
                                                   dim=1, keepdim=True) * math.sqrt(case["cols"]) * leaves["post"]
    if case["gate"]:
        branch = branch * leaves["gate"].reshape(runs, -1).repeat_interleave(case["rows"] // runs, 0)
    total = branch + (leaves["residual"] * leaves["scale"] if case["scale"] else leaves["residual"])
    size = torch.linalg.vector_norm(torch.cat([total, torch.full_like(total[:, :1], math.sqrt(EPS * case["cols"]))], 1), dim=1, keepdim=True)
    normed = total / size * math.sqrt(case["cols"]) * leaves["weight"]
    if case["eight"]:
        return dict(total=total.detach(), values=_eighth(normed.detach()))
    out = dict(out=normed.detach(), total=total.detach())
    if case["train"]:
        names = sorted(leaves)
        grads = torch.autograd.grad((normed, total), [leaves[k] for k in names], (wide["grad_out"], wide["grad_total"]))
        out.update({"d" + k: g for k, g in zip(names, grads)})
    return out


def _exact_adamw(case, state, wide):
    flat, step, (b1, b2) = {k: v.double() for k, v in state["flat"].items()}, FIRST_STEP + 1, BETAS
    g = flat["g"] / LOSS_SCALE
    whole = lambda name: flat[name].view(-1, BLOCK).mul(flat[name + "_scale"].unsqueeze(1)).view(-1)   # noqa: E731
    m, v = (whole("m"), whole("v").square()) if case["bits"] == 8 else (flat["m"], flat["v"])
    m, v = torch.lerp(g, m, b1), torch.lerp(g.square(), v, b2)
    p = flat["p"] * (1 - LR * DECAY) - LR * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + ADAM_EPS)
    out = dict(p=p)
    if "copy" in flat:
        out["copy"] = p
    if "clamped" in flat:
        out["clamped"] = torch.clamp(p, *BOUNDS)
    if case["bits"] == 32:
        out.update(m=m, v=v)
        return out
    # a step of float8_e4m3fn: an eighth of the power of two below a number, 2^-9 at the least; a fraction of a step goes up where it
    # and the dither come to a whole one
    place = torch.arange(BLOCK, device=p.device, dtype=torch.float64)
    first = torch.remainder(place * 0x9E3779B1 + step * 0x6A09E667, 2.0 ** 32)
    for name, value, dither in (("m", m, first), ("v", v.sqrt(), torch.remainder(first + 2.0 ** 31, 2.0 ** 32))):
        rows = value.view(-1, BLOCK)
        largest = rows.abs().max(dim=1).values
        scale = torch.where(largest > 0, torch.exp2(torch.floor(torch.log2(largest)) - 7), 2.0 ** -126)
        size = rows.abs() / scale[:, None]
        unit = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
        codes = torch.floor(size / unit + torch.floor(dither / 4096) / 2.0 ** 20) * unit
        if name == "v":
            codes = torch.where(rows > 0, codes.clamp(min=2.0 ** -9), 0.0)
        out[name] = (codes * torch.sign(rows)).view(-1)
        out[name + "_scale"] = scale
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        each = 2 * size + TYPES[case["grad"]].itemsize + (4 + 4 / BLOCK if case["bits"] == 8 else 16)
        each += (TYPES[case["copy"]].itemsize if case["copy"] != "none" else 0) + (4 if case["clamp"] else 0)
        return dict(bytes=int(n * each), flops=16 * n)
    rows, cols = case["rows"], case["cols"]
    cells = rows * cols
    if case["op"] == "norm":
        # x, residual in, the sum and the norm out; both gradients in, both out
        moved = 3 * size + (2 if case["eight"] else size) + (4 * size if case["train"] else 0)
        around = 1 + case["post"] + case["gate"] + case["scale"]
        return dict(bytes=cells * moved + cols * around * size * (2 if case["train"] else 1), flops=cells * (40 if case["train"] else 12))
    inner, extra = case["inner"], (cols * size if case["bias"] else 0) + (cells * size if case["residual"] else 0)
    if not case["train"]:
        return dict(bytes=(rows + cols) * (inner + 4) + cells * size + extra, flops=2 * cells * inner)
    # x, w, the gradient, bias and residual in; y, dx, dw and the bias's gradient out (the residual's is the gradient itself)
    return dict(bytes=2 * size * (rows * inner + cols * inner + cells) + extra + (cols * size if case["bias"] else 0), flops=6 * cells * inner)
