"""The output projection in 8-bit floating point: ``proj_out`` with e4m3 weights
and one scale for each block of 128.

``Fp8Weight`` holds a weight as checkpoints of this format do: e4m3 values and one
fp32 scale for each 128 ids x 128 values.  ``lm_head_logits_fp8`` quantises the
hidden states of a call, one scale for each row's 128 values, and multiplies on
the tcgen05 tensor cores, each block's sum scaled by both in fp32 (their product
has to be in fp32's range): the counterpart of
:func:`~mapperatorinator_b200.sampling.lm_head_logits` (modeling_varwhisper.py:1583)
and of :func:`~mapperatorinator_b200.int8_head.lm_head_logits_int8`, whose one scale
a row a few large channels coarsen, and which is the faster of the two from a few
hundred rows on.
:meth:`~mapperatorinator_b200.sampling.FusedSampler.step_hidden` takes an
:class:`Fp8Weight` in the weight's place.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .int8_head import DTYPES, launch_on, matrix, same_device

BLOCK = 128


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


class Fp8Weight(NamedTuple):
    """e4m3 weight rows ``q`` [V, d] (row stride a multiple of 16 bytes) and the fp32
    scales [ceil(V / 128), ceil(d / 128)] of their blocks."""

    q: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def from_weight(cls, weight: torch.Tensor) -> "Fp8Weight":
        """Quantises an ``nn.Linear`` weight ``[V, d]``, one scale for each 128 x 128 block."""
        return cls(*quantize_blocks(weight, block_rows=BLOCK))

    def dequantize(self) -> torch.Tensor:
        """The fp32 weight that the blocks stand for."""
        rows, cols = self.q.shape
        scale = self.scale.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
        return self.q.float() * scale


def quantize_blocks(x: torch.Tensor, *, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 values of ``x`` [R, C] and the fp32 scales [ceil(R / block_rows),
    ceil(C / 128)] of its blocks of ``block_rows`` (1 or 128) rows and 128 columns:
    ``scale = max|x| * (1 / 448)`` (the reciprocal and the product rounded to fp32)
    and ``q = x / scale``, rounded to fp32 and to e4m3 (half to even), held to -448 ..
    448.  A block of zeros gives zeros and scale 0; one with a NaN or an infinity
    gives zeros and scale NaN.  The rows of ``q`` start on 16-byte boundaries (it may
    be a view of wider rows)."""
    stride = matrix(x, "x")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x has no columns")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}")
    wide = (cols + 15) // 16 * 16
    q = torch.empty((rows, wide), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((_blocks(rows) if block_rows > 1 else rows, _blocks(cols)), dtype=torch.float32, device=x.device)
    a = N.sized(N.MtrQuantizeBlocksArgs, x=x.data_ptr(), x_row_stride=stride, x_dtype=DTYPES[x.dtype], rows=rows, cols=cols,
                block_rows=block_rows, q=q.data_ptr(), q_row_stride=wide, scale=scale.data_ptr(), scale_row_stride=scale.shape[1])
    launch_on(x.device, N.quantize_blocks_launch, a)
    return q[:, :cols], scale


def lmhead_f8_args(hidden: torch.Tensor, weight_q: torch.Tensor, weight_scale: torch.Tensor,
                   out: torch.Tensor) -> tuple[N.MtrLmHeadF8Args, torch.Tensor | None]:
    """The launch arguments and the workspace they point to (to be kept until the launch)."""
    hs, ws, ls = matrix(hidden, "hidden"), matrix(weight_q, "weight_q", (torch.float8_e4m3fn,)), matrix(out, "logits")
    ss = matrix(weight_scale, "weight_scale", (torch.float32,))
    device = hidden.device
    rows, d = hidden.shape
    vocab = weight_q.shape[0]
    for t, what in ((weight_q, "weight_q"), (weight_scale, "weight_scale"), (out, "logits")):
        same_device(t, device, what)
    if weight_q.shape[1] != d:
        raise ValueError(f"hidden d_model {d} != weight d_model {weight_q.shape[1]}")
    if weight_scale.shape != (_blocks(vocab), _blocks(d)):
        raise ValueError(f"weight_scale must be [{_blocks(vocab)}, {_blocks(d)}]: one scale for each 128 x 128 block")
    if out.shape[0] != rows or out.shape[1] != vocab:
        raise ValueError("logits must be [hidden rows, vocab]")
    if vocab == 1:
        ws = (d + 15) // 16 * 16
    need = N.lmhead_f8_workspace(rows, d, vocab)  # 0 for few rows
    work = hidden.new_empty(need, dtype=torch.uint8) if need else None
    a = N.sized(N.MtrLmHeadF8Args, hidden=hidden.data_ptr(), hidden_row_stride=hs, weight=weight_q.data_ptr(),
                weight_row_stride=ws, weight_scale=weight_scale.data_ptr(), scale_row_stride=ss, logits=out.data_ptr(),
                logits_row_stride=ls, hidden_dtype=DTYPES[hidden.dtype], logits_dtype=DTYPES[out.dtype], rows=rows, d_model=d,
                vocab=vocab, workspace=work.data_ptr() if need else None, workspace_bytes=need)
    return a, work


def lm_head_logits_fp8(hidden: torch.Tensor, weight_q: torch.Tensor, weight_scale: torch.Tensor,
                       out: torch.Tensor | None = None, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``proj_out(hidden)`` with an e4m3 weight: ``[R, V]`` logits from hidden states
    ``[R, d]`` (float32, bfloat16 or float16), weight rows ``[V, d]`` (float8_e4m3fn,
    row stride a multiple of 16 bytes) and the scales of their 128 x 128 blocks.  The
    logits are ``out``, or a new tensor of ``out_dtype``; any of the three dtypes.  Not
    differentiable.  Logits that a wait that gave up left without a value are NaN
    (:func:`~mapperatorinator_b200.sampling.projection_timeouts`)."""
    if out is None:
        if out_dtype not in DTYPES:
            raise TypeError(f"out_dtype {out_dtype} is not supported (float32, bfloat16, float16)")
        out = hidden.new_empty((hidden.shape[0], weight_q.shape[0]), dtype=out_dtype)
    a, work = lmhead_f8_args(hidden, weight_q, weight_scale, out)
    launch_on(hidden.device, N.lmhead_f8_launch, a)
    return out
