"""Functional SC layer with the reference's interface (utils_functional.py), for the
configurations this build accelerates, all with the LFSR generators and ``legacy=False``:
``forward='1d_bin'`` (OR over input channels and kernel dim 2, binary add over kernel dim 3),
``forward='z_bin'`` (OR over the kernel window, add over input channels) and
``forward='yz_bin'`` (OR over ``z_unit`` input channels and kernel dim 2, add over kernel dim 3
and channel blocks).

Forward values come from the HIP SC kernels (integer counts / stream length); gradients
are those of the reference's floating-point surrogates ``conv2d_or_bin_1d`` / ``_z`` / ``_yz``
(utils_functional.py:235-299), computed by the HIP backward kernels instead of autograd
over two dense convolutions per add group.  The surrogate's own forward is never evaluated: the
reference overwrites its value with the SC result anyway (utils_functional.py:631-634).
"""
from __future__ import annotations

import torch

from . import _native, capi

# Default precision is 8-bit integer, one bit is the sign (utils_functional.py:28)
prec_default = 7


def quantize(input, prec=8):
    """round(x * 2^prec) clamped to +-(2^prec - 1), scaled back (utils_functional.py:33-39)."""
    if input.is_cuda and input.dtype == torch.float32 and input.is_contiguous() and isinstance(prec, int) \
            and 1 <= prec <= 23 and not (torch.is_grad_enabled() and input.requires_grad):
        return capi.quantize(input, prec)   # the same values from one kernel instead of four
    prec_2 = 2 ** prec
    return (input * prec_2).round().clamp(-prec_2 + 1, prec_2 - 1) / prec_2


def quantize_shift(tensor, scale=None, scale_only=False):
    """Power-of-two scale, then 8-bit quantisation of tensor/scale (utils_functional.py:41-57)."""
    if scale_only:
        scale = 2 ** torch.ceil(torch.log2(torch.mean(tensor) * 2))
        return torch.ones_like(tensor) * scale, scale
    if scale is None:
        scale = 2 ** torch.ceil(torch.log2(torch.mean(tensor) * 3))
    q = ((tensor / scale) * 128).round().clamp(-127, 127) / 128
    return q * scale, scale


class _SCConv2dAddPartial(torch.autograd.Function):
    """value: SC count / L  (HIP forward);  gradient: surrogate (HIP backward)."""

    @staticmethod
    def forward(ctx, activation, weight, bit_length, padding, load_unit, load_wait, accumulate="y", z_unit=1,
                load_wait_a=None, generator="lfsr", seed=0, prec=None):
        origin = activation.device
        dev = origin if activation.is_cuda else torch.device("cuda", torch.cuda.current_device())
        x = activation.detach().to(dev, torch.float32).contiguous()
        w = weight.detach().to(dev, torch.float32).contiguous()
        pad = (int(padding[0]), int(padding[1]))
        if activation.is_cuda:
            # sc_extension_cuda.conv2d_add_partial_variable_acc(..., prec_default, load_unit,
            # load_wait_w, False, 2): one wait for both generators (utils_functional.py:497)
            # (:504), and conv2d_add_yz_variable_acc(..., load_wait_w, load_wait_a, False, z_unit) (:508)
            loading = dict(total_width=prec_default, load_width=int(load_unit), load_wait_w=int(load_wait),
                           load_wait_a=int(load_wait if load_wait_a is None else load_wait_a))
        else:
            # host tensors take the reference's CPU entry point, which has no progressive
            # loading (utils_functional.py:493)
            loading = dict(capi.NEUTRAL_LOADING)
        z_unit = max(1, min(int(z_unit), x.shape[1]))
        if generator != "lfsr":
            loading = dict(capi.NEUTRAL_LOADING)  # the random generators have no progressive loading
        desc = capi.make_desc(x.shape, w.shape, int(bit_length), pad, accumulate=accumulate, z_unit=z_unit,
                              generator=generator, seed=seed, **loading)
        values = capi.conv2d_add_partial_values(x, w, desc, int(bit_length))
        ctx.save_for_backward(x, w)
        ctx.accumulate = accumulate
        ctx.z_unit = z_unit
        ctx.pad = pad
        ctx.origin = origin
        ctx.bit_length = int(bit_length)
        ctx.prec = prec
        ctx.act_dtype = activation.dtype
        ctx.w_dtype = weight.dtype
        ctx.w_device = weight.device
        return values.to(origin)

    @staticmethod
    def backward(ctx, grad_out):
        x, w = ctx.saved_tensors
        g = grad_out.detach().to(x.device, torch.float32).contiguous()
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        gx = gw = None
        if need_x or need_w:
            gx, gw = capi.conv2d_add_partial_backward(x, w, g, ctx.bit_length, ctx.pad, need_x, need_w,
                                                      accumulate=ctx.accumulate, z_unit=ctx.z_unit,
                                                      options=capi.operand_options(ctx.prec))
        if gx is not None:
            gx = gx.to(ctx.origin, ctx.act_dtype)
        if gw is not None:
            gw = gw.to(ctx.w_device, ctx.w_dtype)
        return gx, gw, None, None, None, None, None, None, None, None, None, None


def conv2d_generic(activation, weight, padding, stride, **kwargs):
    """Generic SC conv2d layer, same call as the reference's (utils_functional.py:406-634).

    Keyword arguments read: bit_length (128), generator (None), forward ('full_or'), legacy
    (False), load_unit (8), load_wait_w (1), load_wait_a (1), z_unit (1024), prec (None: not known; the bits that activation
    and weight were quantised to, which the backward may take to look for operands of few bits); acc/share are
    accepted and unused on these paths.  Implemented: forward='1d_bin' with generator='lfsr' or,
    on GPU tensors, 'acc'; forward='z_bin' / 'yz_bin' on GPU tensors (the reference sends those to
    its LFSR GPU ops whatever the generator, utils_functional.py:503-510); forward='full_or' on GPU
    tensors (random Bernoulli streams, :511-514); all with legacy=False; anything else raises
    NotImplementedError.
    """
    bit_length = kwargs.get("bit_length", 128)
    generator = kwargs.get("generator", None)
    forward = kwargs.get("forward", "full_or")
    legacy = kwargs.get("legacy", False)
    load_unit = kwargs.get("load_unit", 8)
    load_wait_w = kwargs.get("load_wait_w", 1)
    load_wait_a = kwargs.get("load_wait_a", 1)
    z_unit = kwargs.get("z_unit", 1024)
    prec = kwargs.get("prec", None)
    ok_1d = forward == "1d_bin" and (generator == "lfsr" or (generator == "acc" and activation.is_cuda))
    ok_zyz = forward in ("z_bin", "yz_bin", "full_or") and activation.is_cuda
    if legacy or not (ok_1d or ok_zyz):
        raise NotImplementedError(
            f"conv2d_generic(forward={forward!r}, generator={generator!r}, legacy={legacy}, "
            f"cuda={activation.is_cuda}): this build implements forward='1d_bin' with generator='lfsr' and "
            "(on GPU tensors also 'acc'), and forward='z_bin'/'yz_bin'/'full_or' on GPU tensors, legacy=False")
    if isinstance(stride, int):
        stride = (stride, stride)
    if tuple(stride) != (1, 1):
        raise NotImplementedError("the SC kernels compute stride 1 only (the reference's native code ignores stride)")
    if isinstance(padding, int):
        padding = (padding, padding)
    if forward == "full_or":
        # sc_extension_cuda.conv2d_or_acc: Bernoulli random streams, OR over everything
        # (utils_functional.py:511-514); surrogate conv2d_or_approx (:616-617)
        return _SCConv2dAddPartial.apply(activation, weight, bit_length, tuple(padding), 8, 1, "full", 1, None, "rand",
                                         0, prec)
    if forward == "1d_bin" and generator == "acc":
        # sc_extension_cuda.conv2d_add_partial_acc_acc (utils_functional.py:499-502)
        return _SCConv2dAddPartial.apply(activation, weight, bit_length, tuple(padding), 8, 1, "y", 1, None, "acc", 37,
                                         prec)
    if forward == "z_bin":
        return _SCConv2dAddPartial.apply(activation, weight, bit_length, tuple(padding), load_unit, load_wait_w, "z",
                                         1, None, "lfsr", 0, prec)
    if forward == "yz_bin":
        return _SCConv2dAddPartial.apply(activation, weight, bit_length, tuple(padding), load_unit, load_wait_w,
                                         "yz", z_unit, load_wait_a, "lfsr", 0, prec)
    return _SCConv2dAddPartial.apply(activation, weight, bit_length, tuple(padding), load_unit, load_wait_w, "y", 1, None,
                                     "lfsr", 0, prec)


def sc_counts(activation, weight, bit_length, padding, forward="1d_bin", load_unit=8, load_wait_w=1, load_wait_a=1,
              z_unit=1024):
    """int32 SC counts of one layer without autograd (inference).  ``activation`` is fp32, or
    uint8 holding the 7-bit integers round(x * 128) that the fused layer epilogue emits.  Same
    argument meaning as ``conv2d_generic``'s keywords (utils_functional.py:406-510)."""
    if forward not in ("1d_bin", "z_bin", "yz_bin"):
        raise NotImplementedError(f"sc_counts(forward={forward!r})")
    mode = {"1d_bin": "y", "z_bin": "z", "yz_bin": "yz"}[forward]
    wait_a = load_wait_a if mode == "yz" else load_wait_w
    kw = dict(total_width=prec_default, load_width=int(load_unit), load_wait_w=int(load_wait_w),
              load_wait_a=int(wait_a), accumulate=mode, z_unit=max(1, min(int(z_unit), activation.shape[1])))
    pad = (int(padding[0]), int(padding[1]))
    w = weight.detach().float().contiguous()
    if activation.dtype == torch.uint8:
        return capi.conv2d_add_partial_forward_q7(activation.contiguous(), w, int(bit_length), pad, **kw)
    return capi.conv2d_add_partial_forward(activation.detach().float().contiguous(), w, int(bit_length), pad, **kw)


# ---------------------------------------------------------------- dense layers in 8-bit integers
#
# The SC layers approximate products of 8-bit operands; these compute them exactly, with a scale per row in place of the one
# fixed scale of ``quantize``.  All take GPU tensors (float32, bfloat16 or float16; rows are the last dimension) and run on PyTorch's
# current stream.  The gradients can be taken once: a second derivative raises, as does a forward-mode tangent.

_dense_module = None


def _dense():
    global _dense_module
    if _dense_module is None:
        _dense_module = _native.module("sc_dense")
    return _dense_module


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def quantize_rows(x, values=None):
    """Each row of ``x`` in 8 bits: ``scale = max|row| / 127`` and ``q = round(row * 127 / max|row|)``, half to even.
    Returns (q int8, scale float32 per row, values): ``values`` is ``q * scale`` in the type that the argument names, or None.
    A row of zeros has scale 0, a row with an infinity or NaN scale NaN.  No gradients: see ``linear_q8``."""
    return _dense().quantize_rows(x, values)


def rms_norm_q8(x, weight, residual=None, eps=1e-6, values=None):
    """Root-mean-square norm of ``x + residual`` with 8-bit output: with ``total = x + residual``, the rows of
    ``total / sqrt(mean(total^2) + eps) * weight`` as ``quantize_rows`` has them.  Returns (q, scale, total, values);
    ``total`` is ``x`` where there is no residual, ``values`` is None unless a type is named.

    ``q`` and ``scale`` are for ``matmul_q8`` and carry no gradient.  For training name a type of ``values``: the values
    and ``total`` are differentiable, the rounding passing the gradient through; or take ``norm_linear_q8``."""
    if _wants_grad(x, weight, residual):
        if values is None:
            raise ValueError("rms_norm_q8 under autograd needs the type of values, which carry the gradient (or torch.no_grad())")
        return _dense().rms_norm_q8_grad(x, weight, residual, eps, values)
    return _dense().rms_norm_q8(x, weight, residual, eps, values)


def matmul_q8(q, scale, weight_q, weight_scale, dtype=torch.float32, bias=None, activation=None, residual=None):
    """``y[..., n] = act(scale[...] * weight_scale[n] * sum_k q[..., k] * weight_q[n, k] + bias[n]) + residual[..., n]`` for 8-bit rows with a
    scale each (``quantize_rows``, ``rms_norm_q8``, ``gated_norm_q8``); the integer sum is exact (at most 131071 terms), what follows is
    float32, ``y``, rounded once, of ``dtype``.  ``bias``: (columns,) of any of the three types; ``activation``: None, "relu", "gelu" (z times
    the normal distribution's share below z, to 0.75e-7 of that) or "silu" (z / (1 + exp(-z))); ``residual``: of y's shape and type.  No gradients: see
    ``linear_q8``."""
    if bias is None and activation is None and residual is None:
        return _dense().matmul_q8(q, scale, weight_q, weight_scale, dtype)
    if _wants_grad(bias, residual):
        raise ValueError("matmul_q8 has no gradients: take linear_q8 (or torch.no_grad())")
    return _dense().matmul_q8_epilogue(q, scale, weight_q, weight_scale, dtype, bias, activation, residual)


def linear_q8(x, weight, bias=None, activation=None, residual=None):
    """``act(x @ weight.t() + bias) + residual`` with both operands of the product rounded to 8-bit rows first, in ``x``'s type
    (``matmul_q8`` says what the epilogue takes).  The gradients are those of the product at the rounded operands, passed straight
    through the rounding, as ``Conv2d_Add_Partial`` passes its own.  The upstream gradient, times a scale and the activation's slope, enters them
    with 11 bits where it is bfloat16 and with 23 where it is float16 or float32; the slope of gelu and silu is kept with 11 bits for bfloat16, with
    24 otherwise."""
    if bias is None and activation is None and residual is None:
        return _dense().linear_q8(x, weight)
    return _dense().linear_q8_epilogue(x, weight, bias, activation, residual)


def norm_linear_q8(x, gain, weight, residual=None, eps=1e-6, bias=None, activation=None):
    """The root-mean-square norm of ``x + residual`` with 8-bit output (``rms_norm_q8``, weight ``gain``) and its
    product with ``weight`` rounded to 8-bit rows, with bias and activation (``matmul_q8``): (y, x + residual), differentiable (once)
    in all tensors."""
    return _dense().norm_linear_q8(x, gain, weight, residual, eps, bias, activation)


# ---------------------------------------------------------------- distillation

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def distill_topk(logits, top_logits, top_index, temperature=1.0, reduction="mean"):
    """Divergence of the student's softmax from a teacher's top logits, for training: per row of ``logits`` (rows,
    columns), with p the softmax of ``top_logits / temperature`` over the row's entries and q the softmax of ``logits /
    temperature`` over all columns, ``temperature^2 * sum_k p_k (log p_k - log q[top_index_k])``.

    ``top_logits`` and ``top_index`` (int32 or int64) are (rows, entries), at most 4096 entries; an index outside the columns (-1)
    marks an absent entry, and a row without entries has loss and gradient 0.  ``reduction``: "mean" over all rows, "sum" or
    "none".  The loss is float32; the gradient, which can be taken once, goes to ``logits`` only (the teacher is
    fixed)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    return _dense().distill_topk(logits, top_logits, top_index, temperature, _REDUCTIONS[reduction])


# ---------------------------------------------------------------- between two blocks

def gated_norm(x, residual, weight, post_weight=None, gate=None, residual_scale=None, eps=1e-6):
    """The norm behind a block, its gate, the scaled residual and the norm in front of the next block, in one pass: for a block's output
    ``x`` and the stream ``residual`` beside it, with ``rms(v) = sqrt(mean(v^2) + eps)`` over the last dimension::

        m = x / rms(x) * post_weight                    (without post_weight: m = x)
        total = residual_scale * residual + gate * m    (each 1 where it is None)
        out = total / rms(total) * weight

    Returns (out, total) in ``x``'s type, which all tensors have; sums and factors are float32.  ``weight``, ``post_weight`` and
    ``residual_scale`` are (columns,), ``gate`` (columns,) or of x's dimensions with ones behind the leading ones that it has: (samples,
    1, columns) for x of (samples, tokens, columns).  Differentiable (once) in all of them."""
    return _dense().gated_norm(x, residual, weight, post_weight, gate, residual_scale, eps,
                               _wants_grad(x, residual, weight, post_weight, gate, residual_scale))


def gated_norm_q8(x, residual, weight, post_weight=None, gate=None, residual_scale=None, eps=1e-6, values=None):
    """``gated_norm`` with its ``out``, before it is rounded to a type, as ``quantize_rows`` has it, for the 8-bit products of a served network: (q,
    scale, total, values), ``values`` None unless a type is named.  No gradients: train with ``gated_norm_linear_q8``."""
    if _wants_grad(x, residual, weight, post_weight, gate, residual_scale):
        raise ValueError("gated_norm_q8 has no gradients: take gated_norm (or torch.no_grad())")
    return _dense().gated_norm_q8(x, residual, weight, post_weight, gate, residual_scale, eps, values)


def gated_norm_linear_q8(x, residual, gain, weight, post_weight=None, gate=None, residual_scale=None, eps=1e-6, bias=None, activation=None):
    """``gated_norm_q8`` (its weight is ``gain``) and the product of its rows with ``weight`` rounded to 8-bit rows, with bias and activation
    (``matmul_q8``): (y, total), differentiable (once) in all tensors.  The norm's output goes from float32 to 8 bits, as it does in a served
    network: both give the same bits."""
    return _dense().gated_norm_linear_q8(x, residual, gain, weight, post_weight, gate, residual_scale, eps, bias, activation)


# ---------------------------------------------------------------- optimiser step

def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, grad_scale=1.0, scales=None,
               copies=None, clamped=None, bounds=(-1.0, 0.999)):
    """One AdamW step on lists of contiguous GPU tensors (those of a parameter of its shape), in place, in fp32 operations whatever their types: with
    t = ``step`` and g = ``grads * grad_scale``::

        m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        params = params (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    ``params`` and ``grads`` are float32, bfloat16 or float16.  States of 32 bits: ``exp_avg`` and ``exp_avg_sq`` hold m and v
    (float32).  States of 8 bits, where ``scales`` is a pair of lists: ``exp_avg`` holds m, ``exp_avg_sq`` the root of v, both
    as ``torch.float8_e4m3fn`` numbers times a power of two (``torch.float8_e8m0fnu``) for each 256 elements of the flattened tensor; numbers
    between two codes go up or down so that the mean over steps is right.  All-zero states (scales too) are those of no step.

    ``step`` is the number of this step, from 1 on, or an int64 GPU tensor of one element that holds the number of steps done, which
    the call counts up: that is the form to record in a graph.  ``copies``: tensors that receive the new parameters, before their rounding, in a
    type of their own.  ``clamped``: float32 tensors (or None) that receive them clamped to ``bounds``."""
    counted = step if torch.is_tensor(step) else None
    _dense().adamw_step(params, grads, exp_avg, exp_avg_sq, 0 if counted is not None else step, counted, lr, betas[0], betas[1], eps,
                        weight_decay, grad_scale, scales[0] if scales else None, scales[1] if scales else None, copies, clamped, *bounds)
