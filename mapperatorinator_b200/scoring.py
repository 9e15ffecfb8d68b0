"""Scores of given tokens: log probabilities, entropy and top alternatives.

``token_logprobs`` reads each row of logits once and says what the row's
softmax gives to a token, how uncertain it is and which tokens it prefers --
what a served step reports beside its tokens
(:class:`~mapperatorinator_b200.sampling.FusedSampler` with
``token_logprobs=n``), and what a training loss is made of: the log
probabilities, the entropy, the log-sum-exp and the alternatives' log
probabilities are differentiable with respect to the logits, without a stored
softmax.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .int8_head import DTYPES, launch_on, matrix, no_tangent, same_device


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives for R rows."""

    logprobs: torch.Tensor | None  # [R] float32, None without tokens
    entropy: torch.Tensor          # [R] float32, nats
    lse: torch.Tensor              # [R] float32
    top_ids: torch.Tensor          # [R, n] int64, -1 where there are fewer alternatives
    top_logprobs: torch.Tensor     # [R, n] float32
    stats: torch.Tensor            # [R, 4] float32, for token_logprobs_backward


def _tokens(tokens: torch.Tensor | None, logits: torch.Tensor) -> torch.Tensor | None:
    if tokens is None:
        return None
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens dtype {tokens.dtype} is not supported (int64, int32)")
    if tokens.shape != logits.shape[:1]:
        raise ValueError(f"tokens must have one id per row ({logits.shape[0]})")
    same_device(tokens, logits.device, "tokens")
    return tokens.contiguous()


def _forward(logits: torch.Tensor, tokens: torch.Tensor | None, top_n: int, temperature: float,
             status: torch.Tensor | None) -> TokenLogprobs:
    stride = matrix(logits, "logits")
    rows, vocab = logits.shape
    device = logits.device
    if status is not None:
        if status.dtype != torch.int32 or status.shape != (rows,) or not status.is_contiguous():
            raise ValueError(f"status must be a contiguous int32 vector of {rows} elements")
        same_device(status, device, "status")
    n = int(top_n)
    if not 0 <= n <= N.MAX_TOP_N:
        raise ValueError(f"top_n must be 0 .. {N.MAX_TOP_N}")
    f32 = torch.float32
    stats = logits.new_empty((rows, 4), dtype=f32)
    entropy = logits.new_empty(rows, dtype=f32)
    lse = logits.new_empty(rows, dtype=f32)
    logprobs = logits.new_empty(rows, dtype=f32) if tokens is not None else None
    top_ids = logits.new_empty((rows, n), dtype=torch.int64)
    top_logprobs = logits.new_empty((rows, n), dtype=f32)
    a = N.sized(N.MtrLogprobArgs, logits=logits.data_ptr(), logits_row_stride=stride, logits_dtype=DTYPES[logits.dtype],
                tokens_dtype=N.IDS_I32 if tokens is not None and tokens.dtype == torch.int32 else N.IDS_I64,
                rows=rows, vocab=vocab, top_n=n, temperature=float(temperature), out_entropy=entropy.data_ptr(),
                out_lse=lse.data_ptr(), out_stats=stats.data_ptr())
    if tokens is not None:
        a.tokens, a.out_logprobs = tokens.data_ptr(), logprobs.data_ptr()
    if n:
        a.out_top_ids, a.out_top_logprobs = top_ids.data_ptr(), top_logprobs.data_ptr()
    if status is not None:
        a.out_status = status.data_ptr()
    launch_on(device, N.logprob_launch, a)
    return TokenLogprobs(logprobs, entropy, lse, top_ids, top_logprobs, stats)


def _grad_input(g: torch.Tensor | None, shape, device, what: str) -> torch.Tensor | None:
    if g is None:
        return None
    if g.dtype != torch.float32 or tuple(g.shape) != tuple(shape):
        raise ValueError(f"{what} must be float32 of shape {tuple(shape)}")
    same_device(g, device, what)
    return g.contiguous()  # sums and means hand in expanded scalars


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor | None, result: TokenLogprobs, *,
                            grad_logprobs: torch.Tensor | None = None, grad_entropy: torch.Tensor | None = None,
                            grad_lse: torch.Tensor | None = None, grad_top_logprobs: torch.Tensor | None = None,
                            temperature: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``token_logprobs(logits, tokens, ...)`` with respect to the
    logits, from that call's ``result`` and the gradients of its outputs (None:
    zeros).  This is what autograd runs; called directly it needs no autograd
    graph, so it can be captured in a CUDA graph.  ``logits``, ``tokens`` and
    ``temperature`` are the forward call's; ``out`` has the logits' shape and
    dtype and must not overlap them.  Itself not differentiable."""
    no_tangent("token log probabilities", logits, grad_logprobs, grad_entropy, grad_lse, grad_top_logprobs)
    stride = matrix(logits, "logits")
    rows, vocab = logits.shape
    device = logits.device
    tokens = _tokens(tokens, logits)
    stats, top_ids = result.stats, result.top_ids
    n = top_ids.shape[1] if grad_top_logprobs is not None else 0
    if stats.dtype != torch.float32 or stats.shape != (rows, 4) or not stats.is_contiguous():
        raise ValueError(f"result.stats must be a contiguous float32 [{rows}, 4] tensor")
    if n and (top_ids.dtype != torch.int64 or top_ids.shape[0] != rows or not top_ids.is_contiguous()):
        raise ValueError(f"result.top_ids must be a contiguous int64 tensor of {rows} rows")
    for t, what in ((stats, "result.stats"), (top_ids, "result.top_ids")):
        same_device(t, device, what)
    if grad_logprobs is not None and tokens is None:
        raise ValueError("grad_logprobs needs the tokens")
    gl = _grad_input(grad_logprobs, (rows,), device, "grad_logprobs")
    ge = _grad_input(grad_entropy, (rows,), device, "grad_entropy")
    gz = _grad_input(grad_lse, (rows,), device, "grad_lse")
    gt = _grad_input(grad_top_logprobs, top_ids.shape, device, "grad_top_logprobs")
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=device)
    elif out.dtype != logits.dtype or out.shape != logits.shape:
        raise ValueError("out must have the logits' shape and dtype")
    out_stride = matrix(out, "out")
    same_device(out, device, "out")
    return _launch_backward(logits, stride, tokens, stats, top_ids, n, gl, ge, gz, gt, temperature, out, out_stride)


def _launch_backward(logits, stride, tokens, stats, top_ids, n, gl, ge, gz, gt, temperature, out, out_stride) -> torch.Tensor:
    """The launch of token_logprobs_backward; every argument has been checked."""
    rows, vocab = logits.shape
    a = N.sized(N.MtrLogprobGradArgs, logits=logits.data_ptr(), logits_row_stride=stride,
                logits_dtype=DTYPES[logits.dtype],
                tokens_dtype=N.IDS_I32 if tokens is not None and tokens.dtype == torch.int32 else N.IDS_I64,
                rows=rows, vocab=vocab, top_n=n, temperature=float(temperature), stats=stats.data_ptr(),
                grad_logits=out.data_ptr(), grad_row_stride=out_stride)
    if tokens is not None:
        a.tokens = tokens.data_ptr()
    if gl is not None:
        a.g_logprobs = gl.data_ptr()
    if ge is not None:
        a.g_entropy = ge.data_ptr()
    if gz is not None:
        a.g_lse = gz.data_ptr()
    if n:
        a.top_ids, a.g_top = top_ids.data_ptr(), gt.data_ptr()
    launch_on(logits.device, N.logprob_grad_launch, a)
    return out


class _TokenLogprobs(torch.autograd.Function):
    """The differentiable outputs; the whole result is left in ``hold``."""

    @staticmethod
    def forward(ctx, logits, tokens, top_n, temperature, status, hold):
        r = _forward(logits, tokens, top_n, temperature, status)
        ctx.save_for_backward(logits, tokens, r.stats, r.top_ids)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        hold.append(r)
        return r.logprobs, r.entropy, r.lse, r.top_logprobs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_lse, g_top):
        logits, tokens, stats, top_ids = ctx.saved_tensors
        if g_logprobs is None and g_entropy is None and g_lse is None and g_top is None:
            return None, None, None, None, None, None
        # autograd has given the gradients their outputs' types and shapes
        gl, ge, gz, gt = (g if g is None else g.contiguous() for g in (g_logprobs, g_entropy, g_lse, g_top))
        n = top_ids.shape[1] if gt is not None else 0
        stride, grad = matrix(logits, "logits"), logits.new_empty(logits.shape)
        _launch_backward(logits, stride, tokens, stats, top_ids, n, gl, ge, gz, gt, ctx.temperature, grad, logits.shape[1])
        return grad, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top_n: int = 0, temperature: float = 1.0,
                   status: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under ``softmax(logits / temperature)``, with
    the entropy, the log-sum-exp and the ``top_n`` most probable ids of each row.

    ``logits`` is ``[R, V]`` (float32, bfloat16 or float16, any row stride >= V),
    ``tokens`` ``[R]`` int64 or int32, or None for the entropy, log-sum-exp and
    alternatives alone; ``top_n`` is at most 32, ``temperature`` at most 2^100.
    Results are float32.

    - Masked ids (-inf) have probability 0, add nothing to the entropy and are
      never alternatives: where a row has fewer ids left the missing ones read
      id -1 and log probability -inf.  Equal logits are listed in id order.
    - A token below 0 (a padded position, e.g. -100) has log probability 0 and
      no gradient; so has one >= V, which also sets the row's ``bad_id`` bit.
    - A row with every id masked reads log probability and lse -inf, entropy 0,
      gradient 0; a row with a NaN or +inf reads NaN.

    ``status`` (int32 ``[R]``) receives the row bits that
    :func:`~mapperatorinator_b200.sampling.row_status_report` reads.  Gradients
    flow from ``logprobs``, ``entropy``, ``lse`` and ``top_logprobs`` to the
    logits (once, in reverse mode; not through ``top_ids``)."""
    no_tangent("token log probabilities", logits)
    tokens = _tokens(tokens, logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        hold: list = []
        logprobs, entropy, lse, top_logprobs = _TokenLogprobs.apply(logits, tokens, top_n, temperature, status, hold)
        return TokenLogprobs(logprobs, entropy, lse, hold[0].top_ids, top_logprobs, hold[0].stats)
    return _forward(logits, tokens, top_n, temperature, status)
