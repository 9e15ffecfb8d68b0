"""Distillation from a teacher's top logits.

A draft model learns from what a larger model prefers at each position: the ids
and log probabilities that :func:`~mapperatorinator_b200.scoring.token_logprobs`
reports as ``top_ids`` and ``top_logprobs``.  ``distillation_loss`` is the
Kullback-Leibler divergence of the student's softmax from them, differentiable
with respect to the student's logits; ``distillation_loss_and_grad`` gives losses
and gradient from one reading of the logits and without an autograd graph.
"""

from __future__ import annotations

import torch

from . import _native as N
from .int8_head import DTYPES, launch_on, matrix, no_tangent, same_device


def _args(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, temperature: float, tail: bool,
          status: torch.Tensor | None) -> N.MtrDistillArgs:
    stride = matrix(logits, "logits")
    rows, vocab = logits.shape
    device = logits.device
    ids_stride = matrix(teacher_ids, "teacher_ids", (torch.int64, torch.int32))
    lps_stride = matrix(teacher_logprobs, "teacher_logprobs", (torch.float32,))
    for t, what in ((teacher_ids, "teacher_ids"), (teacher_logprobs, "teacher_logprobs")):
        same_device(t, device, what)
        if t.shape[0] != rows:
            raise ValueError(f"{what} must have one row per row of logits ({rows})")
    n = teacher_ids.shape[1]
    if teacher_logprobs.shape[1] != n:
        raise ValueError(f"teacher_logprobs must have {n} columns, as teacher_ids")
    if not 1 <= n <= N.MAX_TEACHER_IDS:
        raise ValueError(f"a row must have 1 .. {N.MAX_TEACHER_IDS} teacher ids")
    if status is not None:
        if status.dtype != torch.int32 or status.shape != (rows,) or not status.is_contiguous():
            raise ValueError(f"status must be a contiguous int32 vector of {rows} elements")
        same_device(status, device, "status")
    a = N.sized(N.MtrDistillArgs, logits=logits.data_ptr(), logits_row_stride=stride, teacher_ids=teacher_ids.data_ptr(),
                ids_row_stride=ids_stride, teacher_logprobs=teacher_logprobs.data_ptr(), logprobs_row_stride=lps_stride,
                logits_dtype=DTYPES[logits.dtype], ids_dtype=N.IDS_I32 if teacher_ids.dtype == torch.int32 else N.IDS_I64,
                rows=rows, vocab=vocab, n=n, tail=int(bool(tail)), temperature=float(temperature))
    if status is not None:
        a.out_status = status.data_ptr()
    return a


def _grad_losses(g: torch.Tensor | None, logits: torch.Tensor) -> torch.Tensor | None:
    if g is None:
        return None
    if g.dtype != torch.float32 or g.shape != logits.shape[:1]:
        raise ValueError(f"grad_losses must be a float32 vector of {logits.shape[0]} elements")
    same_device(g, logits.device, "grad_losses")
    return g.contiguous()


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_ids, teacher_logprobs, temperature, tail, status):
        a = _args(logits, teacher_ids, teacher_logprobs, temperature, tail, status)
        loss = logits.new_empty(logits.shape[0], dtype=torch.float32)
        stats = logits.new_empty((logits.shape[0], 2), dtype=torch.float64)
        a.out_loss, a.stats = loss.data_ptr(), stats.data_ptr()
        launch_on(logits.device, N.distill_launch, a)
        ctx.save_for_backward(logits, teacher_ids, teacher_logprobs, stats)
        ctx.temperature, ctx.tail = temperature, tail
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, teacher_ids, teacher_logprobs, stats = ctx.saved_tensors
        a = _args(logits, teacher_ids, teacher_logprobs, ctx.temperature, ctx.tail, None)
        g, grad = g.contiguous(), logits.new_empty(logits.shape)
        a.g_loss, a.stats, a.grad_logits, a.grad_row_stride = g.data_ptr(), stats.data_ptr(), grad.data_ptr(), logits.shape[1]
        launch_on(logits.device, N.distill_launch, a)
        return grad, None, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      temperature: float = 1.0, tail: bool = False, status: torch.Tensor | None = None) -> torch.Tensor:
    """Losses ``[R]`` (float32) of the student ``q = softmax(logits / temperature)``
    against a teacher's top ids.

    ``logits`` is ``[R, V]`` (float32, bfloat16 or float16, any row stride >= V),
    ``teacher_ids`` ``[R, n]`` int64 or int32 and ``teacher_logprobs`` ``[R, n]``
    float32, n at most 128.  They are constants; a temperature of the teacher's is
    applied by whoever computed them, and no loss is multiplied by T^2.

    - ``tail=False``: ``p`` is the teacher's distribution over its ids alone,
      renormalised (so logits serve as well as log probabilities);
      ``loss = sum_j p_j (log p_j - log q_j)``.
    - ``tail=True``: what the teacher did not list is one more outcome, of
      probability ``1 - sum p`` against the student's mass outside the ids.  (A rest
      below 2^-20 is the rounding of the given log probabilities and counts as 0.)
    - An id below 0 is no entry; so is one >= V, which also sets the row's ``bad_id``
      bit; a log probability of -inf is probability 0.  A row without entries (a
      padded position; with ``tail=False`` also one whose entries all have probability
      0) has loss 0 and gradient 0, whatever its logits hold.  An id that is given
      twice is two entries.
    - Where the student has no mass and the teacher has some the loss is +inf; a row
      with a NaN or +inf reads NaN; one with every logit masked has gradient 0.

    ``status`` (int32 ``[R]``) receives the row bits that
    :func:`~mapperatorinator_b200.sampling.row_status_report` reads.  Gradients flow
    to the logits (once, in reverse mode).  A step that is to be captured in a CUDA
    graph takes :func:`distillation_loss_and_grad`: autograd's backward must not be
    captured while an eager graph of the same leaves is alive."""
    no_tangent("distillation losses", logits, teacher_logprobs)
    if torch.is_grad_enabled():
        if teacher_logprobs.requires_grad:
            raise ValueError("teacher_logprobs must not require a gradient: the teacher is a constant")
        if logits.requires_grad:
            return _Loss.apply(logits, teacher_ids, teacher_logprobs, temperature, tail, status)
    a = _args(logits, teacher_ids, teacher_logprobs, temperature, tail, status)
    loss = logits.new_empty(logits.shape[0], dtype=torch.float32)
    a.out_loss = loss.data_ptr()
    launch_on(logits.device, N.distill_launch, a)
    return loss


def distillation_loss_and_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor,
                               grad_losses: torch.Tensor | None = None, *, temperature: float = 1.0, tail: bool = False,
                               out: torch.Tensor | None = None,
                               status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The losses of :func:`distillation_loss` and the gradient of
    ``sum_r grad_losses[r] loss[r]`` (None: ones) with respect to the logits, from
    one reading of the logits.  No autograd graph is needed or made, so a training
    step can be captured in a CUDA graph.  The gradient is ``out`` or a new tensor;
    ``out`` has the logits' shape and dtype and must not overlap them."""
    no_tangent("distillation losses", logits, teacher_logprobs, grad_losses)
    a = _args(logits, teacher_ids, teacher_logprobs, temperature, tail, status)
    g = _grad_losses(grad_losses, logits)
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty(logits.shape)
    elif out.dtype != logits.dtype or out.shape != logits.shape:
        raise ValueError("out must have the logits' shape and dtype")
    a.grad_row_stride = matrix(out, "out")
    same_device(out, logits.device, "out")
    loss = logits.new_empty(logits.shape[0], dtype=torch.float32)
    a.out_loss, a.grad_logits = loss.data_ptr(), out.data_ptr()
    if g is not None:
        a.g_loss = g.data_ptr()
    launch_on(logits.device, N.distill_launch, a)
    return loss, out
