"""Criteria of the reference's training loop, computed by fused HIP kernels (log-softmax, loss and gradient in
one pass over fp32 logits; linear_cross_entropy / LinearCrossEntropy take the features and the head's weight instead, for label sets
whose fp32 logits and their gradient are too large to hold).

Mirrors main.py:926-935 (criterion choice: timm SoftTargetCrossEntropy when mixup is on, timm
LabelSmoothingCrossEntropy(smoothing) when smoothing > 0, else nn.CrossEntropyLoss) and the inline knowledge
distillation classes main.py:836-851 (StudentWithDistillation) and main.py:939-970 (DistillationLoss), duplicated in
test_kd.py:43-88.
"""
from __future__ import annotations

import os

import torch
import torch.nn as nn

from . import ops
from ._lib import EPI_BIAS_F32, VitkError

bf16, f32 = torch.bfloat16, torch.float32


def _as_logits(x):
    if not x.is_cuda:
        raise VitkError("criterion: logits must be on the GPU; the fused loss kernels are the only implementation")
    if x.dtype != torch.float32:
        x = x.float()
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.reshape(x.shape[0], -1).contiguous()
    return x


class _FusedLoss(torch.autograd.Function):
    """mean over the batch of a per-row loss; the kernel already produced d(mean loss)/d(logits)."""

    @staticmethod
    def forward(ctx, logits, kind, arg0, arg1):
        B = logits.shape[0]
        want = logits.requires_grad and torch.is_grad_enabled()
        if kind == "label":
            rows, dl = ops.xent_label(logits, arg0, arg1, 1.0 / B, want_grad=True)
        elif kind == "soft":
            rows, dl = ops.xent_soft(logits, arg0, 1.0 / B, want_grad=True)
        else:   # "kd": arg0 = teacher logits, arg1 = temperature; 'batchmean' = sum over rows / B
            rows, dl = ops.kd_kl(logits, arg0, arg1, 1.0 / B, want_grad=True)
        ctx.dl = dl
        return rows.mean()

    @staticmethod
    def backward(ctx, go):
        dl, ctx.dl = ctx.dl, None
        return dl * go, None, None, None


class LabelSmoothingCrossEntropy(nn.Module):
    """timm.loss.LabelSmoothingCrossEntropy: mean_b[(1-eps) * nll_b + eps * mean_c(-logp_bc)]"""

    def __init__(self, smoothing: float = 0.1):
        super().__init__()
        assert smoothing < 1.0
        self.smoothing = smoothing

    def forward(self, x, target):
        return _FusedLoss.apply(_as_logits(x), "label", target.contiguous(), float(self.smoothing))


class CrossEntropyLoss(nn.Module):
    """nn.CrossEntropyLoss() with integer targets (main.py:934, engine.py:341)"""

    def forward(self, x, target):
        return _FusedLoss.apply(_as_logits(x), "label", target.contiguous(), 0.0)


class SoftTargetCrossEntropy(nn.Module):
    """timm.loss.SoftTargetCrossEntropy: mean_b sum_c -t_bc * logp_bc"""

    def forward(self, x, target):
        t = target
        if t.dtype != torch.float32 or t.stride(-1) != 1:
            t = t.float().contiguous()
        return _FusedLoss.apply(_as_logits(x), "soft", t, None)


def _bf16_rows(t):
    """a bf16 matrix with contiguous, 16-byte aligned rows holding t's values (t itself where it is one)"""
    t = t.detach()
    if t.numel() == 0:
        return t.to(bf16)
    if t.dtype == f32 or t.stride(-1) != 1 or (t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1])):
        t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return ops.cast_f32_to_bf16(t) if t.dtype == f32 else t


def _times(g, go):
    """g * go in place of g; the upstream scalar go stays fp32 where g is bf16, so that the product is what is rounded and not the scalar"""
    if g is None or g.numel() == 0:
        return g
    if g.dtype == bf16 and g.dim() == 2:
        return ops.rowscale(g, go.reshape(1).float(), g.shape[0], out=g)
    if g.dtype == f32:
        return g.mul_(go.float())
    return g.copy_(g.float() * go.float())          # bf16 times a scalar on the GPU would round the scalar first


class _LinearXent(torch.autograd.Function):
    """The loss and, where anything needs them, its gradients in one call of ops.linear_xent; backward multiplies them by the upstream scalar."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, smoothing, ignore_index, reduction, want):
        wtype = weight.dtype
        grads = [n for n, need in zip(("x", "weight", "bias"), ctx.needs_input_grad) if need]
        r = ops.linear_xent(_bf16_rows(x), _bf16_rows(weight), target, None if bias is None else bias.detach(), smoothing=smoothing,
                            ignore_index=ignore_index, reduction=reduction, want_grad=want, dweight_dtype=wtype if wtype in (bf16, f32) else None, grads=grads)
        ctx.grads = (r.dx, r.dweight, r.dbias) if want else None
        ctx.xtype = x.dtype
        return r.loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        if ctx.grads is None:
            raise VitkError("linear_cross_entropy: backward was called a second time (the gradients are handed over, not kept)")
        (dx, dw, db), ctx.grads = ctx.grads, None
        dx = _times(dx, go)
        return None if dx is None else dx.to(ctx.xtype), _times(dw, go), _times(db, go), None, None, None, None, None


def linear_cross_entropy(x, weight, target, bias=None, smoothing: float = 0.0, ignore_index: int = -100, reduction: str = "mean"):
    """cross entropy of the logits x @ weight.T + bias, of which 2 bytes each are held for a block of rows at a time (ops.linear_xent): x [..., D], weight [V, D] (bf16, or fp32
    masters, which are rounded to bf16 for the products as every linear of this package does), bias [V], target [...] int64.
    Differentiable in x, weight and bias, once.  reduction 'mean' (over the targets that are not ignore_index) or 'sum'."""
    if x.dim() < 1 or tuple(x.shape[:-1]) != tuple(target.shape):
        raise VitkError(f"linear_cross_entropy: target must be {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    for t, n in ((x, "x"), (weight, "weight")):
        if t.dtype not in (bf16, f32):
            raise VitkError(f"linear_cross_entropy: {n} must be bfloat16 or float32, got {t.dtype}")
        ops._here(t, f"linear_cross_entropy: {n}")
    want = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
    return _LinearXent.apply(x.reshape(-1, x.shape[-1]), weight, bias, target.reshape(-1), float(smoothing), int(ignore_index), reduction, want)


class LinearCrossEntropy(nn.Module):
    """A classification head and its criterion in one: owns weight [num_classes, in_features] and bias (fp32 masters, timm's head
    initialisation), takes the features instead of the logits.  For label sets so large that the logits and their gradient are what fills
    the memory: 21 843 classes, or the vocabulary of a token-prediction objective over every position.  As a criterion of train_one_epoch it is
    clipped together with the model and averaged over its ranks; its parameters belong into the optimizer beside the model's
    (optimizer.add_param_group), itself into evaluate, save_model and auto_load_model (criterion=...).  A weight average (utils.ModelEma)
    does not cover it."""

    takes_features = True           # train_one_epoch: the model's output is not a matrix of logits

    def __init__(self, in_features: int, num_classes: int, bias: bool = True, smoothing: float = 0.0, ignore_index: int = -100, reduction: str = "mean"):
        super().__init__()
        if in_features < 8 or in_features % 8 or num_classes < 1:
            raise VitkError(f"LinearCrossEntropy: in_features must be a multiple of 8, num_classes positive, got {in_features}, {num_classes}")
        if not 0.0 <= smoothing <= 1.0 or reduction not in ("mean", "sum"):
            raise VitkError(f"LinearCrossEntropy: smoothing outside [0, 1] or unknown reduction: {smoothing}, {reduction!r}")
        self.smoothing, self.ignore_index, self.reduction = float(smoothing), int(ignore_index), reduction
        self.weight = nn.Parameter(torch.empty(num_classes, in_features))
        nn.init.trunc_normal_(self.weight, std=0.02)
        self.bias = nn.Parameter(torch.zeros(num_classes)) if bias else None

    def forward(self, x, target):
        return linear_cross_entropy(x, self.weight, target, self.bias, self.smoothing, self.ignore_index, self.reduction)

    @torch.no_grad()
    def logits(self, x):
        """fp32 logits [rows, num_classes] of features [rows, in_features], for evaluation and prediction: no gradient, and as large as they are"""
        V, D = self.weight.shape
        if x.dim() != 2 or x.shape[1] != D:
            raise VitkError(f"LinearCrossEntropy.logits: expected features [rows, {D}], got {tuple(x.shape)}")
        ops._here(x, "LinearCrossEntropy.logits: features")
        if x.shape[0] == 0:
            return x.new_empty((0, V), dtype=f32)
        w, b, room = self.weight.detach(), self.bias, (V + 3) // 4 * 4           # the product wants a multiple of 4 classes
        if room != V:
            w = torch.nn.functional.pad(w, (0, 0, 0, room - V))
        bias = torch.zeros(room, dtype=f32, device=x.device)
        if b is not None:
            bias[:V] = b.detach()
        return ops.gemm_nt(_bf16_rows(x), _bf16_rows(w), epilogue=EPI_BIAS_F32, bias=bias)[:, :V].contiguous()


class DistillationLoss(nn.Module):
    """(1-alpha) * base(student, y) + alpha * T^2 * KL_batchmean(softmax(teacher/T) || log_softmax(student/T))
    when given (student_logits, teacher_logits); base(outputs, y) otherwise (main.py:939-970)."""

    def __init__(self, base_criterion, alpha: float = 0.7, temperature: float = 4.0):
        super().__init__()
        self.base_criterion, self.alpha, self.temperature = base_criterion, alpha, temperature

    def forward(self, outputs, targets):
        if isinstance(outputs, tuple):
            student_logits, teacher_logits = outputs
            ce = self.base_criterion(student_logits, targets)
            kd = _FusedLoss.apply(_as_logits(student_logits), "kd", _as_logits(teacher_logits.detach()), float(self.temperature))
            return (1 - self.alpha) * ce + self.alpha * kd
        return self.base_criterion(outputs, targets)


class StudentWithDistillation(nn.Module):
    """train mode: (student(x), teacher(x) under no_grad); eval mode: student(x)  (main.py:836-851)"""

    def __init__(self, student_model, teacher_model):
        super().__init__()
        self.student = student_model
        self.teacher = teacher_model

    def forward(self, x):
        if not (self.training and self.teacher is not None):
            return self.student(x)
        # The two forward passes do not depend on each other.  Where the student has a side stream (the one its weight-gradient
        # GEMMs use in backward, idle now), the teacher runs there: each model's GEMMs fill the compute units that the other's
        # last tile rounds leave empty.  The teacher's activations are allocated under that stream, so its allocator pool
        # hands them on in that stream's order; only the logits cross over, behind the event.
        side = self.student._wgrad_stream() if (x.is_cuda and hasattr(self.student, "_wgrad_stream")
                                                and os.environ.get("VITK_KD_OVERLAP", "1") != "0") else None
        if side is None:
            student_logits = self.student(x)
            with torch.no_grad():
                teacher_logits = self.teacher(x)
            return student_logits, teacher_logits
        ready = torch.cuda.Event()
        ready.record()                                   # x is complete once everything queued so far has run
        side.wait_event(ready)
        with torch.cuda.stream(side), torch.no_grad():
            teacher_logits = self.teacher(x)
            done = torch.cuda.Event()
            done.record(side)
        student_logits = self.student(x)
        torch.cuda.current_stream().wait_event(done)     # the loss reads the teacher's logits; x may be released after this
        return student_logits, teacher_logits
