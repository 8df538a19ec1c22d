"""Distillation from a teacher's top logits: the student's distribution over the
whole vocabulary against the teacher's over the k tokens it kept.

    from memoryefficientclip_amd import TopKDistillationLoss, token_log_probs
    t = token_log_probs(teacher_logits, tokens, top_k=32)            # once, or stored with the data
    loss = TopKDistillationLoss(temperature=2.0)(student_logits, t.top_tokens, t.top_log_probs)

Loss of a position:  T^2 KL(q || p),  q = softmax(teacher / T) over the k entries,
p = softmax(student / T) over the vocabulary.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from . import _vocab as _v

_REDUCTIONS = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}


def _check(student_logits, teacher_tokens, teacher_logits):
    _v.check_gpu("student_logits", student_logits)
    _v.check_gpu("teacher_tokens", teacher_tokens, student_logits.device)
    _v.check_gpu("teacher_logits", teacher_logits, student_logits.device)
    _v.refuse_graph_capture()
    _v.refuse_make_fx()
    _v.check_float("student_logits", student_logits)
    _v.check_float("teacher_logits", teacher_logits)
    _v.check_tokens("teacher_tokens", teacher_tokens)
    shape, teacher_shape = student_logits.shape, teacher_tokens.shape
    if teacher_shape != teacher_logits.shape:
        raise ValueError(f"teacher_tokens {tuple(teacher_shape)} and teacher_logits {tuple(teacher_logits.shape)} differ "
                         f"in shape")
    if min(len(shape), len(teacher_shape)) < 1 or shape[:-1] != teacher_shape[:-1]:
        raise ValueError(f"student_logits {tuple(shape)} and teacher_tokens {tuple(teacher_shape)} need the same "
                         f"positions")
    vocab, k = shape[-1], teacher_shape[-1]
    if not 1 <= vocab <= _lib.MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {_lib.MAX_VOCAB} tokens, got {vocab}")
    if not 1 <= k <= _lib.MAX_TEACHER_K:
        raise ValueError(f"a position needs 1 to {_lib.MAX_TEACHER_K} teacher entries, got {k}")


def _loss(logits, rows, teacher_tokens, teacher_logits, temperature, weight, reduction, need):
    """The loss, and with `need` what the backward needs; logits and their rows as ``rows_of`` has them."""
    code, teacher_code, token_bytes = _v.code_of(logits), _v.code_of(teacher_logits), teacher_tokens.element_size()
    teacher_tokens, teacher_logits = teacher_tokens.contiguous(), teacher_logits.contiguous()
    shape, k, dev = logits.shape, teacher_tokens.shape[-1], logits.device
    vocab = shape[-1]
    loss = torch.empty(shape[:-1] if reduction == _lib.REDUCE_NONE else (), dtype=torch.float32, device=dev)
    state = torch.empty(2 * rows[0] + 1, dtype=torch.float32, device=dev)
    # The gradient for grad_output 1 is made while the row is at hand: the
    # logits are read once for loss and gradient.  fp16 programs scale their
    # losses, so there grad_output is not 1 and the backward makes it.
    dx = None
    if need and reduction != _lib.REDUCE_NONE and logits.dtype != torch.float16:
        dx = torch.empty(shape, dtype=logits.dtype, device=dev)
    lib = _lib.load()
    nbytes = lib.mec_distill_workspace_bytes(rows[0], vocab, k, code, int(dx is not None))
    rc = _v.launch(dev.index, nbytes, lambda ws, stream: lib.mec_distill_forward(
        logits.data_ptr(), *rows, vocab, code, teacher_tokens.data_ptr(), token_bytes, teacher_logits.data_ptr(),
        teacher_code, k, temperature, weight, reduction, loss.data_ptr(), state.data_ptr(),
        None if dx is None else dx.data_ptr(), ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_distill_forward", rc)
    kept = ((logits, rows, teacher_tokens, teacher_logits, state) + (() if dx is None else (dx,)),
            (vocab, code, token_bytes, teacher_code, k, temperature, weight, reduction))
    return loss, kept


def _logits_grad(ctx, grad_output):
    held, rows, teacher_tokens, teacher_logits, state, *dx = _v.saved_logits(ctx)
    vocab, code, token_bytes, teacher_code, k, temperature, weight, reduction = ctx.mec
    go = grad_output.contiguous()
    # The forward's gradient is handed out once, since its new owner may change it: as a
    # tensor of its own on the same memory (autograd copies one that others hold, and
    # takes a change of it for one of what is saved).
    made, ctx.made = ctx.made, False
    dx = dx[0].data if made else held.new_empty(held.shape)
    lib = _lib.load()
    rc = _v.launch(held.device.index, 0, lambda ws, stream: lib.mec_distill_backward(
        held.data_ptr(), *rows, vocab, code, teacher_tokens.data_ptr(), token_bytes, teacher_logits.data_ptr(),
        teacher_code, k, temperature, weight, reduction, state.data_ptr(), go.data_ptr(), int(made), dx.data_ptr(),
        stream))
    if rc:
        raise _lib.error("mec_distill_backward", rc)
    return dx, None, None, None, None, None, None


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, teacher_tokens, teacher_logits, temperature, weight, reduction):
        need = True
        if rows is None:
            _check(logits, teacher_tokens, teacher_logits)
            need = ctx.needs_input_grad[0]
            logits, _, rows = _v.rows_of(logits)
        loss, kept = _loss(logits, rows, teacher_tokens, teacher_logits, temperature, weight, reduction, need)
        _v.save_logits(ctx, *kept[0])
        ctx.mec, ctx.made = kept[1], len(kept[0]) > 5
        return loss

    backward = _v.backward_of(_logits_grad)


class TopKDistillationLoss(nn.Module):
    """``forward(student_logits [..., V], teacher_tokens [..., k], teacher_logits [..., k])``.

    ``teacher_logits`` are the teacher's logits or log probabilities of
    ``teacher_tokens`` (both mean the same to the softmax over them); an entry
    with a token < 0 is none, and a position with no entry has loss 0, gradient
    0 and no part in the mean.  ``reduction``: "mean" over the positions that
    have a teacher, "sum" or "none"; fp32.  ``weight`` multiplies the loss.
    Gradients flow to the student's logits only.

    With "mean" and "sum" the forward leaves the gradient for ``grad_output`` 1
    beside the loss (fp32 and bf16 logits), so that a training step reads the logits
    once; with any other ``grad_output`` the backward makes it anew.  To
    weight the loss against another, use ``weight``; to have the loss alone,
    ``torch.no_grad()``.
    """

    def __init__(self, temperature=1.0, reduction="mean", weight=1.0):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
        self.temperature = _v.check_temperature(temperature)
        self.reduction = reduction
        self.weight = float(weight)
        if not math.isfinite(self.weight):
            raise ValueError(f"weight must be finite, got {weight}")

    def forward(self, student_logits, teacher_tokens, teacher_logits):
        _check(student_logits, teacher_tokens, teacher_logits)
        reduction = _REDUCTIONS[self.reduction]
        if student_logits.numel() == 0:
            # no position: the graph's link to the logits
            return student_logits.sum(-1, dtype=torch.float32) if reduction == _lib.REDUCE_NONE else \
                student_logits.sum(dtype=torch.float32)
        student_logits, _, rows = _v.rows_of(student_logits)
        args = (teacher_tokens, teacher_logits.detach(), self.temperature, self.weight, reduction)
        if _v.wants_autograd(student_logits):
            # (a trace calls this again, with other inputs)
            return _DistillFn.apply(student_logits, None if _v.is_tracing() else rows, *args)
        return _loss(student_logits, rows, *args, False)[0]


__all__ = ["TopKDistillationLoss"]
