"""The SC networks of the reference's training script restated on this build's layer modules:
the 4-layer CNN (network.py:126-190, ``CONV_tiny_add_partial``) and VGG-16 (network.py:12-124,
``VGG16_add_partial``), and the bookkeeping of one training step (utils_own.py:81-114).  The
reference's LeNet (``CONV_minimal_add_partial``) is not restated: it builds on a layer class that
does not exist in the reference (``utils_class.Linear_Or``, network.py:204-206).
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import utils_class

# loss scale of the reference's training loop (utils_own.py:18, :81)
SCALE_FACTOR = 128


class CONV_tiny_add_partial(nn.Module):
    """conv 3->32 k5 p2 @32x32, BN, AvgPool2, Hardtanh(0,1); 32->32 k5 p2 @16x16; 32->64 k5 p2
    @8x8; conv 64->classes k4 p0 @4x4 as the classifier; BN1d.  Per-layer stream length is
    2**err[i]; load_unit / load_wait are the progressive-loading settings per layer."""

    def __init__(self, num_classes=10, c_ins=3, uniform=False, generator="lfsr", sc_compute="1d_bin", legacy=False,
                 relu=False):
        super().__init__()
        self.bn1 = utils_class.BatchNorm2d_fixed(32)
        self.bn2 = utils_class.BatchNorm2d_fixed(32)
        self.bn3 = utils_class.BatchNorm2d_fixed(64)
        self.bn4 = utils_class.BatchNorm1d_fixed(num_classes)
        self.conv1 = utils_class.Conv2d_Add_Partial(c_ins, 32, kernel_size=5, padding=2, bias=False)
        self.conv2 = utils_class.Conv2d_Add_Partial(32, 32, kernel_size=5, padding=2, bias=False)
        self.conv3 = utils_class.Conv2d_Add_Partial(32, 64, kernel_size=5, padding=2, bias=False)
        self.fc1 = utils_class.Conv2d_Add_Partial(64, num_classes, kernel_size=4, padding=0, bias=False)
        self.tanh = nn.Hardtanh(0, 1)
        self.pool = nn.AvgPool2d(2)
        self.err = [7, 7, 7, 7]
        self.z_unit = [3, 3, 4, 4]
        self.load_unit = [2, 2, 2, 2]
        self.load_wait_w = [2, 2, 2, 2]
        # the reference's forward reads `load_wait`, which its training script sets from the
        # command line (main_conv.py:182); the default there is 2 per layer
        self.load_wait = [2, 2, 2, 2]
        self.num_classes = num_classes
        self.generator = generator
        self.compute = sc_compute
        self.legacy = legacy
        self.relu = relu
        # training mode on the GPU with the LFSR kernels: run every conv + batch norm + pool +
        # hardtanh block as one fused autograd node (same values; gradients to fp32 rounding)
        self.fused_blocks = False
        # batch statistics of the fused blocks: False = from exact integer sums of the counts (one HIP kernel,
        # independent of any reduction order), True = PyTorch's two float reductions, as BatchNorm*_fixed runs
        # them (utils_class.py:52-56): bit-identical to the module chain
        self.fused_torch_stats = False
        if uniform:
            self.conv1.weight_org *= 2
            self.conv2.weight_org *= 2
            self.conv1.weight.data *= 2
            self.conv2.weight.data *= 2

    def _sc(self, conv, x, i, wait_w_index=None):
        j = i if wait_w_index is None else wait_w_index
        return conv(x, err=self.err[i], forward=self.compute, generator=self.generator, z_unit=2 ** self.z_unit[i],
                    legacy=self.legacy, load_unit=self.load_unit[i], load_wait_w=self.load_wait[j],
                    load_wait_a=self.load_wait[i])

    def _fusable(self, x):
        return (self.fused_blocks and self.training and x.is_cuda and not self.legacy and self.generator == "lfsr"
                and self.compute in ("1d_bin", "z_bin", "yz_bin"))

    def _fused(self, conv, bn, x, i, j, **tail):
        return utils_class.sc_conv_block(conv, bn, x, err=self.err[i], forward=self.compute,
                                         z_unit=2 ** self.z_unit[i], load_unit=self.load_unit[i],
                                         load_wait_w=self.load_wait[j], load_wait_a=self.load_wait[i],
                                         torch_stats=self.fused_torch_stats, weight_ready=True, **tail)

    def _block(self, conv, bn, x, i):
        if self._fusable(x):
            return self._fused(conv, bn, x, i, i, relu=self.relu)
        x = bn(self._sc(conv, x, i))
        if self.relu:
            x = F.relu(x)
        return self.tanh(self.pool(x))

    def forward(self, x_in, target=None):
        if self._fusable(x_in):
            # the four layers' weight quantisation (utils_class.py:33) in one launch
            utils_class.quantize_weights([self.conv1, self.conv2, self.conv3, self.fc1])
        x = self._block(self.conv1, self.bn1, x_in, 0)
        x = self._block(self.conv2, self.bn2, x, 1)
        x = self._block(self.conv3, self.bn3, x, 2)
        # the classifier layer takes the third layer's weight wait (network.py:186)
        if self._fusable(x):
            y = self._fused(self.fc1, self.bn4, x, 3, 2, relu=False, pool=False, hardtanh=False, quant7=False)
            return y.view(-1, self.num_classes)
        x = self._sc(self.fc1, x, 3, wait_w_index=2)
        return self.bn4(x.view(-1, self.num_classes))


    # ---------------------------------------------------------------- fused inference path
    def train(self, mode=True):
        self._fused_state = None  # parameters may change: drop the cached inference state
        return super().train(mode)

    @torch.no_grad()
    def prepare_fused(self):
        """Cache what an inference forward does not need to recompute: per layer the weight streams
        of the 7-bit-quantised weights and the quantised per-channel affine of its fixed batch
        norm on the running statistics.  Call again after changing parameters or settings."""
        if self.legacy or self.generator != "lfsr" or self.compute not in ("1d_bin", "z_bin", "yz_bin"):
            raise NotImplementedError("forward_fused runs the LFSR kernels only")
        from . import capi, utils_functional as uf
        layers = [(self.conv1, self.bn1, 0, 0), (self.conv2, self.bn2, 1, 1), (self.conv3, self.bn3, 2, 2),
                  (self.fc1, self.bn4, 3, 2)]  # (conv, bn, layer index, index of its weight wait: network.py:186)
        mode = {"1d_bin": "y", "z_bin": "z", "yz_bin": "yz"}[self.compute]
        state = []
        for conv, bn, i, j in layers:
            conv.weight.data = uf.quantize(conv.weight_org, prec=7)
            w = conv.weight.data.float().contiguous()
            wait_w = self.load_wait[j]
            kw = dict(bit_length=2 ** self.err[i], padding=(int(conv.padding[0]), int(conv.padding[1])),
                      total_width=uf.prec_default, load_width=int(self.load_unit[i]), load_wait_w=int(wait_w),
                      load_wait_a=int(self.load_wait[i] if mode == "yz" else wait_w), accumulate=mode,
                      z_unit=max(1, min(2 ** self.z_unit[i], w.shape[1])))
            w_n, b_n = utils_class._fixed_affine(bn, None, bn.running_mean, bn.running_var)
            # the weight stream buffer is generated at the first forward: its stream words do not
            # depend on the input, but what else the buffer carries depends on the layer's geometry
            state.append(dict(w=w, w_shape=tuple(w.shape), kw=kw, wgt=None, wgt_for=None,
                              w_n=w_n.float().contiguous(), b_n=b_n.float().contiguous()))
        self._fused_state = state
        self._fused_graph = None

    def _fused_eager(self, x):
        from . import capi
        last = len(self._fused_state) - 1
        for i, st in enumerate(self._fused_state):
            d = capi.make_desc(x.shape, st["w_shape"], **st["kw"])
            if st["wgt_for"] != tuple(x.shape):
                st["wgt"], st["wgt_for"] = capi.weight_streams(st["w"], d), tuple(x.shape)
            counts = capi.conv2d_add_partial_from_streams(capi.act_streams(x, d), st["wgt"], d)
            L = st["kw"]["bit_length"]
            if i == last:
                logits, _ = capi.layer_epilogue(counts, L, st["w_n"], st["b_n"], relu=False, pool=False,
                                                hardtanh=False, quant7=False)
                return logits.view(-1, self.num_classes)
            _, x = capi.layer_epilogue(counts, L, st["w_n"], st["b_n"], relu=self.relu, want_act=False, want_q7=True)

    @torch.no_grad()
    def forward_fused(self, x_in, graph=False):
        """Inference forward with one fused epilogue kernel per layer in place of the element-wise
        op chain (fixed batch norm on the running statistics, relu, AvgPool2, Hardtanh, the next
        layer's 7-bit quantisation): layers hand each other uint8 7-bit integers, which the
        activation stream generator reads directly, and weight streams come from the cache of
        ``prepare_fused``.  Same logits, bit for bit, as ``forward`` in eval mode.  ``graph=True``
        records the launches of one forward into a HIP graph per input shape and replays it."""
        if self.training:
            raise RuntimeError("forward_fused is the inference path: call model.eval() first")
        from . import utils_functional as uf
        if getattr(self, "_fused_state", None) is None:
            self.prepare_fused()
        x = uf.quantize(x_in.detach().float(), prec=7).contiguous()
        if not graph:
            return self._fused_eager(x)
        g = self._fused_graph
        if g is None or g["x"].shape != x.shape:
            static_x = x.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # warm the allocator and the kernels outside the capture
                self._fused_eager(static_x)
            torch.cuda.current_stream().wait_stream(side)
            cg = torch.cuda.CUDAGraph()
            with torch.cuda.graph(cg):
                out = self._fused_eager(static_x)
            g = self._fused_graph = dict(x=static_x, out=out, graph=cg)
        g["x"].copy_(x)
        g["graph"].replay()
        return g["out"].clone()


class VGG16_add_partial(nn.Module):
    """VGG-16 for SC (network.py:12-124): thirteen 3x3 SC convolutions in five groups
    (2, 2, 3, 3, 3 layers; AvgPool2 and Dropout2d after each group), a 1x1 SC convolution as the
    classifier, fixed batch norm + Hardtanh(0,1) after every layer.  err / z_unit / load_unit /
    load_wait hold one value per group plus one for the classifier; with ``half_pool`` the layer
    in front of a pooling uses half the group's stream length (not below 2**5).  Same attribute
    names as the reference, hence the same ``state_dict`` keys."""

    GROUPS = ((1, 2), (3, 4), (5, 6, 7), (8, 9, 10), (11, 12, 13))
    WIDTHS = (64, 128, 256, 512, 512)

    def __init__(self, uniform=False, sc_compute="1d_bin", generator="lfsr", legacy=False, half_pool=True):
        super().__init__()
        c_in = 3
        for group, width in zip(self.GROUPS, self.WIDTHS):
            for i in group:
                setattr(self, f"conv{i}", utils_class.Conv2d_Add_Partial(c_in, width, kernel_size=3, padding=1,
                                                                         bias=False))
                c_in = width
        for g in range(1, 6):
            setattr(self, f"drop{g}", nn.Dropout2d())
        self.fc1 = utils_class.Conv2d_Add_Partial(512, 10, kernel_size=1, padding=0, bias=False)
        self.pool = nn.AvgPool2d(2)
        for group, width in zip(self.GROUPS, self.WIDTHS):
            for i in group:
                setattr(self, f"bn{i}", utils_class.BatchNorm2d_fixed(width))
        self.bnfc1 = utils_class.BatchNorm1d_fixed(10)
        self.tanh = nn.Hardtanh(0, 1)
        self.err = [7, 7, 7, 7, 7, 7]
        self.z_unit = [5, 5, 5, 5, 5, 5]
        self.load_unit = [2, 2, 2, 2, 2, 2]
        self.load_wait = [2, 2, 2, 2, 2, 2]
        self.generator = generator
        self.compute = sc_compute
        self.legacy = legacy
        self.half_pool = half_pool
        # training mode on the GPU with the LFSR kernels: every conv + batch norm + [pool] + hardtanh
        # block as one fused autograd node (same values; gradients to fp32 rounding)
        self.fused_blocks = False
        if min(self.err) < 4:
            uniform = True
        if uniform:
            for mod in self.modules():
                if isinstance(mod, nn.Conv2d):
                    mod.weight.data.uniform_()
                    mod.weight_org.uniform_()

    def _sc(self, conv, x, g, err):
        return conv(x, err=err, forward=self.compute, generator=self.generator, z_unit=2 ** self.z_unit[g],
                    legacy=self.legacy, load_unit=self.load_unit[g], load_wait_w=self.load_wait[g],
                    load_wait_a=self.load_wait[g])

    def _fused(self, conv, bn, x, g, err, **tail):
        return utils_class.sc_conv_block(conv, bn, x, err=err, forward=self.compute, z_unit=2 ** self.z_unit[g],
                                         load_unit=self.load_unit[g], load_wait_w=self.load_wait[g],
                                         load_wait_a=self.load_wait[g], **tail)

    def forward(self, x):
        pool_offset = 1 if self.half_pool else 0
        fuse = (self.fused_blocks and self.training and x.is_cuda and not self.legacy and self.generator == "lfsr"
                and self.compute in ("1d_bin", "z_bin", "yz_bin"))
        for g, group in enumerate(self.GROUPS):
            for i in group:
                last = i == group[-1]
                err = max(self.err[g] - pool_offset, 5) if last else self.err[g]
                conv, bn = getattr(self, f"conv{i}"), getattr(self, f"bn{i}")
                if fuse:
                    # a dropout follows the group's last layer: its input must stay unquantised
                    x = self._fused(conv, bn, x, g, err, pool=last, quant7=not last)
                    continue
                x = bn(self._sc(conv, x, g, err))
                if last:
                    x = self.pool(x)
                x = self.tanh(x)
            x = getattr(self, f"drop{g + 1}")(x)
        if fuse:
            return self._fused(self.fc1, self.bnfc1, x, 5, self.err[5], pool=False, hardtanh=False,
                               quant7=False).view(-1, 10)
        x = self._sc(self.fc1, x, 5, self.err[5]).view(-1, 10)
        return self.bnfc1(x)


class PatchMLP_q8(nn.Module):
    """Residual network of dense 8-bit layers on image patches: every patch of ``patch`` x ``patch`` pixels is a row; blocks of
    norm, widening, activation and narrowing; the rows' mean through a last norm and layer.  All products are exact 8-bit ones
    (``utils_class.Linear_Q8``), so it serves as the teacher of an SC network (``python -m geo_amd.main_distill``).  ``gated``: each block's
    output is normed and gated before it joins the stream (``utils_class.GatedNormLinear_Q8``, which the layer behind the block is, behind the last
    one the head: every row goes through it, and the logits are their rows' mean); ``bias``: the blocks' layers have one.  Not in the
    reference."""

    def __init__(self, num_classes=10, c_in=3, patch=4, width=256, hidden=1024, depth=4, activation="relu", gated=False, bias=False):
        super().__init__()
        self.patch = patch
        self.gated = gated
        self.embed = utils_class.Linear_Q8(c_in * patch * patch, width)
        inner = dict(bias=bias, activation=activation)
        self.up = nn.ModuleList((utils_class.GatedNormLinear_Q8 if gated and i else utils_class.NormLinear_Q8)(width, hidden, **inner)
                                for i in range(depth))
        self.down = nn.ModuleList(utils_class.Linear_Q8(hidden, width, bias=bias) for _ in range(depth))
        self.head = (utils_class.GatedNormLinear_Q8 if gated and depth else utils_class.NormLinear_Q8)(width, num_classes)

    def _load_from_state_dict(self, state_dict, prefix, *args):
        head = self.head
        if isinstance(head, utils_class.GatedNormLinear_Q8) and prefix + "head.gain" in state_dict and prefix + "head.gate" not in state_dict:
            # saved when the last block was not gated: as it was
            self.head = utils_class.NormLinear_Q8(head.weight.shape[1], head.weight.shape[0]).to(head.weight).train(head.training)
        super()._load_from_state_dict(state_dict, prefix, *args)

    def __setstate__(self, state):
        super().__setstate__(state)
        if "gated" not in state:   # pickled when the relu was the network's own
            self.gated = False
            for up in self.up:
                up.activation = "relu"

    def prepare(self):
        """Round all weights for inference (``Linear_Q8.prepare``)."""
        for layer in self.modules():
            if isinstance(layer, utils_class.Linear_Q8):
                layer.prepare()

    def forward(self, images):
        n, c, h, w = images.shape
        p = self.patch
        if h % p or w % p:
            raise ValueError(f"images of {h} x {w} have no whole patches of {p} x {p}")
        rows = images.reshape(n, c, h // p, p, w // p, p).permute(0, 2, 4, 1, 3, 5).reshape(n, h // p * (w // p), c * p * p)
        y, total = self.embed(rows), None
        for up, down in zip(self.up, self.down):
            wide, total = up(y, total)
            y = down(wide)
        if isinstance(self.head, utils_class.GatedNormLinear_Q8):
            return self.head(y, total)[0].mean(1)
        logits, _ = self.head((y if total is None else total + y).mean(1))
        return logits


def make_param_copies(model):
    """Full-precision master copies the optimiser updates (main_conv.py:203-213)."""
    return [p.detach().clone().float().requires_grad_(True) for p in model.parameters()]


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with all tensors of a step in one kernel (``utils_functional.adamw_step``), states in 32 bits or in
    8.  Parameters are contiguous GPU tensors of float32, bfloat16 or float16; gradients of any of these types.

    ``capturable=True`` counts the steps on the GPU, for steps that are recorded into a graph (``GraphedTrainStep``), where the learning rate
    is recorded with them.  Parameters whose first step was the same are counted together until a step has no gradient for some of them:
    the others are counted apart from there on.  A recorded step cannot part them, nor can any step after one of them all was recorded, whose
    graph counts them together: both are refused, and a step like it is to be made before.  ``apply_update`` hands it the unscaling of the
    gradients and the copies into the parameters as well."""

    _in_graph = ()   # counters that recorded steps count

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, capturable=False):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def add_param_group(self, param_group):
        options = {**self.defaults, **param_group}
        if options["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {options['state_bits']}")
        if not (options["lr"] >= 0 and options["eps"] >= 0 and options["weight_decay"] >= 0 and all(0 <= b < 1 for b in options["betas"])):
            raise ValueError("lr, eps and weight_decay must not be negative, betas in [0, 1)")
        super().add_param_group(param_group)

    def _fresh(self, p, group, step):
        like = lambda n, dtype: torch.zeros(n, dtype=dtype, device=p.device)   # noqa: E731
        state = dict(step=step)
        if group["state_bits"] == 8:
            blocks = (p.numel() + 255) // 256
            state.update(exp_avg=like(p.shape, torch.float8_e4m3fn), exp_avg_sq=like(p.shape, torch.float8_e4m3fn),
                         avg_scale=like(blocks, torch.float8_e8m0fnu), sq_scale=like(blocks, torch.float8_e8m0fnu))
        else:
            state.update(exp_avg=like(p.shape, torch.float32), exp_avg_sq=like(p.shape, torch.float32))
        return state

    def _count_apart(self, group, stepping, recorded):
        """Of parameters that are counted together and do not all make this step, those that do receive a counter of their own."""
        together = {}
        for p in group["params"]:
            state = self.state.get(p)
            if state:
                together.setdefault(id(state["step"]), []).append(p)
        for params in together.values():
            those = [p for p in params if id(p) in stepping]
            if 0 < len(those) < len(params):
                counter = self.state[those[0]]["step"]
                if recorded:   # (every replay would part them anew)
                    raise RuntimeError("a step of some of the parameters that are counted together cannot be recorded: make one like it before")
                if any(counter is c for c in self._in_graph):
                    raise RuntimeError("a step of some of the parameters that are counted together, in a recorded step too: make it before that is recorded")
                counter = counter.clone()
                for p in those:
                    self.state[p]["step"] = counter

    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0, grads=None, copies=None, clamped=None, bounds=(-1.0, 0.999)):
        """One step.  ``grads``, ``copies``, ``clamped``: dicts from parameters to tensors; a gradient that is not among them is the
        parameter's own, a parameter without one stays as it is."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        from . import utils_functional as uf
        recorded = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if recorded and not all(g["capturable"] for g in self.param_groups):
            raise RuntimeError("AdamW(capturable=True) is the one whose steps can be recorded: others count them on the host")
        for group in self.param_groups:
            # parameters that have made the same number of steps; those counted on the GPU, that are counted together
            rows, counters = {}, {}
            stepping = [(p, g) for p in group["params"] if (g := (grads or {}).get(p, p.grad)) is not None]
            if group["capturable"]:
                self._count_apart(group, {id(p) for p, _ in stepping}, recorded)
            for p, g in stepping:
                if g.is_sparse:
                    raise RuntimeError("AdamW takes no sparse gradients")
                state = self.state[p]
                if not state:
                    if recorded:   # (every replay would begin anew)
                        raise RuntimeError("the first step of a parameter, which makes its states, cannot be recorded: do one before")
                    if group["capturable"] and p.device not in counters:
                        counters[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
                    state.update(self._fresh(p, group, counters[p.device] if group["capturable"] else 0))
                step = state["step"] if group["capturable"] else state["step"] + 1
                copy = None if copies is None else copies.get(p)
                # one call per device, number of steps and set of types (those that are not counted on the GPU may mix them)
                types = (p.dtype, g.dtype) if group["capturable"] else None
                key = (p.device, id(step) if group["capturable"] else step, types, None if copy is None else copy.dtype)
                rows.setdefault(key, (step, []))[1].append((p, g.contiguous(), state, copy))
            counted = [step for step, _ in rows.values()]
            if group["capturable"] and len({id(s) for s in counted}) < len(counted):
                raise RuntimeError("AdamW(capturable=True) takes parameters, gradients and copies of one type each in a group")
            for step, row in rows.values():
                states = [state for _, _, state, _ in row]
                uf.adamw_step([p for p, _, _, _ in row], [g for _, g, _, _ in row], [s["exp_avg"] for s in states],
                              [s["exp_avg_sq"] for s in states], step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                              grad_scale, scales=([s["avg_scale"] for s in states], [s["sq_scale"] for s in states])
                              if group["state_bits"] == 8 else None,
                              copies=None if row[0][3] is None else [c for _, _, _, c in row],
                              clamped=None if clamped is None else [clamped.get(p) for p, _, _, _ in row], bounds=bounds)
                if not group["capturable"]:
                    for state in states:
                        state["step"] = step
                elif recorded and not any(step is c for c in self._in_graph):
                    self._in_graph += (step,)
        return loss

    def load_state_dict(self, state_dict):
        """States come back in their own types (the base class would bring them to the parameters'); steps counted on the GPU are
        counted together again where they are equal."""
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, (p, group) in zip(saved, ((p, group) for group in self.param_groups for p in group["params"])):
            if i not in state_dict["state"]:
                continue
            state = self._fresh(p, group, 0)
            for k, v in state_dict["state"][i].items():
                if k == "step":
                    v = int(v)
                elif v.dtype != state[k].dtype or v.shape != state[k].shape:
                    raise ValueError(f"{k} of a parameter of {tuple(p.shape)} does not fit states of {group['state_bits']} bits")
                else:
                    v = v.to(p.device, copy=True)
                state[k] = v
            self.state[p] = state
        for group in self.param_groups:
            together = {}
            for p in group["params"] if group["capturable"] else ():
                if self.state.get(p):
                    step = self.state[p]["step"]
                    self.state[p]["step"] = together.setdefault((p.device, step), torch.full((), step, dtype=torch.int64, device=p.device))


def apply_update(model, optimizer, param_copy):
    """The part of the reference's step that follows ``loss.backward()`` (utils_own.py:98-114): restore
    the full-precision weights, hand the gradients to the master copies and un-scale them, optimiser
    step on the copies, copy back, refresh ``weight_org`` clamped to [-1, 0.999]."""
    # (the reference first copies weight_org back into weight.data; the copy-back from the master copies below
    # overwrites every parameter before anything reads it, so that copy changes nothing and is not launched)
    params = list(model.parameters())
    orgs = {id(m.weight): m.weight_org for m in model.modules() if hasattr(m, "weight_org")}
    if isinstance(optimizer, AdamW) and all(p.is_cuda and p.data.is_contiguous() for p in params) and \
            all(o.dtype == torch.float32 and o.is_contiguous() for o in orgs.values()):
        _apply_adamw(params, orgs, optimizer, param_copy)
        return
    # the per-parameter loops of the reference as multi-tensor calls: one kernel for all gradients,
    # one for all copies
    with_grad = [(master, p) for master, p in zip(param_copy, params) if p.grad is not None]
    for master, p in zip(param_copy, params):
        master.grad = None
    if with_grad:
        scaled = torch._foreach_div([p.grad.data.float() for _, p in with_grad], SCALE_FACTOR)
        for (master, _), g in zip(with_grad, scaled):
            master.grad = g
    optimizer.step()
    if all(p.is_cuda and p.dtype == torch.float32 and p.data.is_contiguous() for p in params):
        # copy back and refresh weight_org, all parameters in one launch
        from . import capi
        capi.copy_back_clamp([master.data for master in param_copy], [p.data for p in params],
                             [orgs.get(id(p)) for p in params], -1, 0.999)
    else:
        torch._foreach_copy_([p.data for p in params], [master.data for master in param_copy])
        for p in params:
            if id(p) in orgs:
                torch.clamp(p.data, -1, 0.999, out=orgs[id(p)])
    optimizer.zero_grad()


def _apply_adamw(params, orgs, optimizer, param_copy):
    """``apply_update`` with the unscaling, the copies back and ``weight_org`` in the optimiser's kernel."""
    known = {id(p) for group in optimizer.param_groups for p in group["params"]}
    stepped = [(master, p) for master, p in zip(param_copy, params) if p.grad is not None and id(master) in known]
    for master in param_copy:
        master.grad = None
    optimizer.step(grads={master: p.grad for master, p in stepped}, grad_scale=1 / SCALE_FACTOR,
                   copies={master: p.data for master, p in stepped},
                   clamped={master: orgs[id(p)] for master, p in stepped if id(p) in orgs}, bounds=(-1, 0.999))
    done = {id(p) for _, p in stepped}
    for master, p in zip(param_copy, params):   # (what is not stepped is copied back all the same: the layers have quantised it)
        if id(p) not in done:
            p.data.copy_(master.data)
            if id(p) in orgs:
                torch.clamp(p.data, -1, 0.999, out=orgs[id(p)])
    optimizer.zero_grad()


def train_step(model, inputs, target, criterion, optimizer, param_copy):
    """One step of the reference's loop (utils_own.py:79-114): scaled loss, backward, then
    ``apply_update``.  Returns the unscaled loss."""
    output = model(inputs)
    loss = criterion(output, target) * SCALE_FACTOR
    for p in model.parameters():
        p.grad = None
    loss.backward()
    apply_update(model, optimizer, param_copy)
    return loss.detach() / SCALE_FACTOR


class GraphedTrainStep:
    """``train_step`` for a fixed batch shape, recorded once into a HIP graph and replayed: the step's ~130
    short launches then cost the host one submission instead of one each (at batch 256 the eager step of the
    4-layer CNN is bound by the host's launch rate, not by the GPU).  Same kernels, same arithmetic, same state:
    weights, master copies, optimiser moments and running statistics live where they did and are updated in
    place by the replayed kernels.

    The optimiser must keep its step count on the device (``torch.optim.Adam(..., capturable=True)``).  Recording
    needs the allocator and the kernels warmed up by real steps; the state they change is put back afterwards
    (model buffers and parameters, master copies, optimiser state), so constructing this object leaves the
    training state as it found it.  The model must be in training mode and stay as it is (same settings, same
    ``fused_blocks``) for as long as the graph is replayed."""

    def __init__(self, model, criterion, optimizer, param_copy, inputs, target, warmup=3):
        import copy
        self.model, self.optimizer, self.param_copy = model, optimizer, param_copy
        self.inputs, self.target = inputs.detach().clone(), target.detach().clone()
        model_state = {k: v.detach().clone() for k, v in model.state_dict().items()}
        masters = [m.detach().clone() for m in param_copy]
        had_state = {id(p) for p in optimizer.state}
        opt_state = copy.deepcopy({id(p): {k: v for k, v in st.items()} for p, st in optimizer.state.items()})
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(max(1, int(warmup))):
                train_step(model, self.inputs.clone(), self.target, criterion, optimizer, param_copy)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            # a second handle on the static batch: the layer re-points its input's .data at the quantised values,
            # which must not re-point self.inputs away from the memory the recorded kernels read
            self.loss = train_step(model, self.inputs.detach(), self.target, criterion, optimizer, param_copy)
        # put the training state back, in place: the graph holds the addresses
        with torch.no_grad():
            now = model.state_dict()
            for k, v in model_state.items():
                now[k].copy_(v)
            for m, saved in zip(param_copy, masters):
                m.copy_(saved)
            for p, st in optimizer.state.items():
                for k, v in st.items():
                    if not torch.is_tensor(v):
                        continue
                    if id(p) in had_state:
                        v.copy_(opt_state[id(p)][k])
                    else:
                        v.zero_()   # a fresh state is all zeros (step count, moments)
        torch.cuda.synchronize()

    def __call__(self, inputs, target):
        """One step on a batch of the recorded shape; returns the (unscaled) loss tensor of that step, which the
        next call overwrites."""
        self.inputs.copy_(inputs)
        self.target.copy_(target)
        self.graph.replay()
        return self.loss
