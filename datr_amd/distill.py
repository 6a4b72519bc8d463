"""Distillation from a teacher of whom each row's top logits were kept (csrc/distill.hip).

The class losses of a teacher-student stage train on thresholded pseudo labels (datr_amd.self_training); this loss trains on
the teacher's distribution instead.  Keeping only a row's largest logits -- `fused.topk_rows(teacher_logits, k)` gives
exactly the pair it takes -- makes a teacher over a large vocabulary affordable to store:

    values, index = topk_rows(teacher_logits, 32)
    loss = (topk_distillation_loss(student_logits, values, index, temperature=2.0) * row_weight).sum()"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _native

MAX_SLOTS = 1024


def _forward(z, teacher, index, tau):
    R, V = z.shape
    loss = torch.empty(R, dtype=torch.float32, device=z.device)
    stats = torch.empty((R, 4), dtype=torch.float32, device=z.device)
    need = int(_native.lib.datr_topk_distill_workspace_floats(_native.DTYPE[z.dtype], R, V))
    ws = torch.empty(need, dtype=torch.float32, device=z.device) if need else None
    with _native.on_device(z.device):
        rc = _native.lib.datr_topk_distill_forward(
            _native.DTYPE[z.dtype], z.data_ptr(), z.stride(0), _native.DTYPE[teacher.dtype], teacher.data_ptr(), index.data_ptr(),
            R, V, teacher.shape[1], tau, loss.data_ptr(), stats.data_ptr(), 0 if ws is None else ws.data_ptr(), need,
            _native.current_stream_ptr(z.device))
    _native.check(rc, "topk_distill_forward")
    return loss, stats


class _TopkDistill(Function):
    @staticmethod
    def forward(ctx, z, teacher, index, tau):
        loss, stats = _forward(z, teacher, index, tau)
        ctx.save_for_backward(z, teacher, index, stats)
        ctx.tau = tau
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        z, teacher, index, stats = ctx.saved_tensors
        R, V = z.shape
        up = upstream if upstream.is_contiguous() else upstream.contiguous()            # the loss is float32, so is this
        dz = torch.empty((R, V), dtype=z.dtype, device=z.device)
        with _native.on_device(z.device):
            rc = _native.lib.datr_topk_distill_backward(
                _native.DTYPE[z.dtype], z.data_ptr(), z.stride(0), _native.DTYPE[teacher.dtype], teacher.data_ptr(),
                index.data_ptr(), R, V, teacher.shape[1], ctx.tau, stats.data_ptr(), up.data_ptr(), dz.data_ptr(),
                _native.current_stream_ptr(z.device))
        _native.check(rc, "topk_distill_backward")
        return dz, None, None, None


def topk_distillation_loss(student: torch.Tensor, teacher: torch.Tensor, index: torch.Tensor,
                           temperature: float = 1.0) -> torch.Tensor:
    """temperature^2 * KL(p || q) per row, float32 [...]: p = softmax(teacher / temperature) over a row's valid slots, q =
    softmax(student / temperature) over all its columns.

    student [..., V] and teacher [..., k]: float32, float16 or bfloat16; index [..., k] int64 / int32: the student's column
    that each slot stands for.  A slot whose index is outside [0, V) is not valid (rows with fewer kept logits: -1); a row
    without a valid slot, or with nothing but -inf in its valid slots, has loss and gradient 0; a NaN in a valid slot gives a
    loss of NaN, and a gradient of NaN in the columns that the row kept; a column named by several slots takes the sum of
    their p.  A student's logit of -inf in a column that the teacher kept (p > 0) makes the row's loss infinite, as the
    formula says, and a row of nothing but -inf has no softmax: NaN.  The temperature is from 1e-30 to 1e18; it
    scales, squared, the roundings of the softmaxes' 32-bit sums and logarithms too, which a large one leaves little beside.
    Differentiable in `student`, once and in reverse mode; the teacher is a constant.  k <= 1024."""
    if student.dtype not in _native.DTYPE or teacher.dtype not in _native.DTYPE:
        name, t = ("student", student) if student.dtype not in _native.DTYPE else ("teacher", teacher)
        raise TypeError(f"topk_distillation_loss: {name} is float32, float16 or bfloat16, got {t.dtype}")
    if index.dtype is not torch.int64 and index.dtype is not torch.int32:
        raise TypeError(f"topk_distillation_loss: index is int64 or int32, got {index.dtype}")
    shape, kept = student.shape, teacher.shape
    if not shape or not kept or index.shape != kept or kept[:-1] != shape[:-1]:
        raise ValueError(f"topk_distillation_loss: student {tuple(shape)}, teacher {tuple(kept)} and index {tuple(index.shape)} do not "
                         "belong together")
    V, k = shape[-1], kept[-1]
    if V < 1:
        raise ValueError("topk_distillation_loss: student has no columns")
    if k > MAX_SLOTS:
        raise NotImplementedError(f"topk_distillation_loss: at most {MAX_SLOTS} kept logits a row, got {k}")
    tau = float(temperature)
    if not 1e-30 <= tau <= 1e18:
        raise ValueError(f"topk_distillation_loss: a temperature from 1e-30 to 1e18, got {temperature}")
    if _native.carries_tangent(student):
        raise RuntimeError("topk_distillation_loss has no forward-mode derivative")
    if not student.is_cuda:
        raise RuntimeError("topk_distillation_loss: Not implemented on the CPU")
    device = student.device
    if teacher.device != device or index.device != device:
        raise ValueError("topk_distillation_loss: student, teacher and index are on different devices")
    z, rows = student, student.numel() // V
    if len(shape) != 2:
        z, teacher, index = z.reshape(rows, V), teacher.reshape(rows, k), index.reshape(rows, k)
    apart, step = z.stride()
    if step != 1 or apart < V:                             # (a single row may have any stride)
        z = z.contiguous().view(rows, V) if rows != 1 else z.contiguous().as_strided((1, V), (V, 1))
    if index.dtype is not torch.int64:
        index = index.to(torch.int64)
    teacher, index = teacher.contiguous(), index.contiguous()
    if student.requires_grad and torch.is_grad_enabled():
        loss = _TopkDistill.apply(z, teacher.detach() if teacher.requires_grad else teacher, index, tau)
    else:
        loss = _forward(z, teacher, index, tau)[0]
    return loss if len(shape) == 2 else loss.view(shape[:-1])
