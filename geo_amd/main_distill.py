"""Distillation of an SC network from a teacher of exact 8-bit layers: trains ``network.PatchMLP_q8``, then an SC network of
``main_conv`` on the divergence from the teacher's top logits (``utils_functional.distill_topk``) mixed with the
cross entropy of the labels.  The command line is main_conv's, with the options below; nothing is saved.  Not in the reference.

    python -m geo_amd.main_distill --dataset SYNTHETIC --err 6666 --epochs 2 --teacher_epochs 2 --top 5 --temperature 4
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.optim as optim

from . import main_conv, network, utils_own
from . import utils_functional as uf


def build_parser():
    p = main_conv.build_parser()
    p.description = "SC CNN trained from an 8-bit teacher's top logits on MI355X"
    p.add_argument("--teacher_epochs", default=10, type=int)
    p.add_argument("--teacher_lr", default=1e-3, type=float)
    p.add_argument("--teacher_optim", default="Adam", choices=("Adam", "AdamW", "AdamW8"), help="AdamW8: states in 8 bits")
    p.add_argument("--teacher_gated", default=0, type=int, help="1: the teacher's blocks are normed and gated behind too, with gelu and biases")
    p.add_argument("--top", default=5, type=int, help="the teacher's logits that the student sees per image")
    p.add_argument("--temperature", default=4.0, type=float)
    p.add_argument("--alpha", default=0.9, type=float, help="weight of the divergence; 1 - alpha: of the labels' cross entropy")
    return p


def _batches(loader, iterations):
    for done, (inputs, target) in enumerate(loader):
        if iterations is not None and done >= iterations:
            return
        yield inputs.cuda(non_blocking=True), target.cuda(non_blocking=True)


def train_teacher(teacher, loader, epochs, lr, iterations=None, optimizer="Adam"):
    """Returns the mean loss of each epoch.  ``optimizer``: "Adam" (PyTorch's), "AdamW" or "AdamW8" (``network.AdamW``)."""
    if optimizer == "Adam":
        optimizer = optim.Adam(teacher.parameters(), lr=lr)
    else:
        optimizer = network.AdamW(teacher.parameters(), lr=lr, state_bits=8 if optimizer == "AdamW8" else 32)
    criterion, losses = nn.CrossEntropyLoss(), []
    teacher.train()
    for _ in range(epochs):
        mean = utils_own.AverageMeter()
        for inputs, target in _batches(loader, iterations):
            loss = criterion(teacher(inputs), target)
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
            mean.update(loss.item(), inputs.size(0))
        losses.append(mean.avg)
    return losses


@torch.no_grad()
def top_logits(teacher, inputs, top):
    """(values, columns) of the ``top`` largest logits of each image, the lowest column first among equals."""
    logits = teacher(inputs)
    order = logits.sort(dim=1, descending=True, stable=True)
    return order.values[:, :top].contiguous(), order.indices[:, :top].to(torch.int32).contiguous()


def distill_step(student, teacher, inputs, target, optimizer, param_copy, top=5, temperature=4.0, alpha=0.9):
    """One training step (``network.train_step``) on ``alpha * distill_topk + (1 - alpha) * cross entropy``; returns the loss."""
    values, columns = top_logits(teacher, inputs, top)

    def criterion(output, target):
        soft = uf.distill_topk(output.float(), values, columns, temperature=temperature)
        return alpha * soft + (1 - alpha) * nn.functional.cross_entropy(output, target)

    # (the SC layers re-point their input's data at the quantised values)
    return network.train_step(student, inputs.detach().clone(), target, criterion, optimizer, param_copy)


def main(argv=None):
    args = build_parser().parse_args(argv)
    torch.manual_seed(args.seed)
    if args.device < 0 or not torch.cuda.is_available():
        raise SystemExit("this build runs on the GPU only: --device must be >= 0 and a GPU must be visible")
    torch.cuda.set_device(args.device)
    trainloader, testloader = main_conv._loaders(args)
    teacher = network.PatchMLP_q8(**(dict(activation="gelu", gated=True, bias=True) if args.teacher_gated else {})).cuda()
    teacher_losses = train_teacher(teacher, trainloader, args.teacher_epochs, args.teacher_lr, args.iterations, args.teacher_optim)
    teacher.eval()
    teacher.prepare()
    print("Teacher: loss per epoch " + " ".join(f"{v:.4f}" for v in teacher_losses))
    student = main_conv.build_model(args).cuda()
    param_copy = network.make_param_copies(student)
    optimizer = optim.Adam(param_copy, lr=args.lr)
    history = []
    for epoch in range(args.epochs):
        student.train()
        mean = utils_own.AverageMeter()
        for inputs, target in _batches(trainloader, args.iterations):
            loss = distill_step(student, teacher, inputs, target, optimizer, param_copy, args.top, args.temperature, args.alpha)
            mean.update(loss.item(), inputs.size(0))
        _, p1, p5 = utils_own.validate(testloader, student, nn.CrossEntropyLoss(), epoch, iteration=args.iterations)
        history.append(dict(epoch=epoch, loss=mean.avg, val_prec1=p1, val_prec5=p5))
        print(f"Epoch: {epoch}\tLoss {mean.avg:.4f}\tPrec@1 {p1:.3f}\tPrec@5 {p5:.3f}")
    return dict(teacher_losses=teacher_losses, history=history)


if __name__ == "__main__":
    main()
