"""The output projection in 8-bit integers: ``proj_out`` with int8 weights.

``quantize_rows`` turns rows into int8 with one fp32 scale each (the weight's
rows once, at load time); ``lm_head_logits_int8`` quantises the hidden states of
a call the same way, multiplies on the tcgen05 tensor cores with exact int32
sums and scales the sums by both: the counterpart of
:func:`~mapperatorinator_b200.sampling.lm_head_logits`
(modeling_varwhisper.py:1583) with half the weight bytes.
:meth:`~mapperatorinator_b200.sampling.FusedSampler.step_hidden` takes an
:class:`Int8Weight` in the weight's place.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}


def launch_on(device: torch.device, launch, *args) -> None:
    """``launch(*args, stream)`` on ``device``'s current stream, with the device made current for it."""
    if device.index == torch._C._cuda_getDevice():
        launch(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            launch(*args, torch._C._cuda_getCurrentRawStream(device.index))


def matrix(t: torch.Tensor, what: str, dtypes=DTYPES) -> int:
    """Checks a 2-D CUDA tensor with unit column stride; returns its row stride in elements."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} dtype {t.dtype} is not supported ({', '.join(str(d)[6:] for d in dtypes)})")
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"{what} must be a 2-D tensor with unit column stride")
    # a single row's stride means nothing and may be anything
    return stride[0] if shape[0] > 1 else max(shape[1], 1)


def same_device(t: torch.Tensor, device: torch.device, what: str) -> None:
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")


class Int8Weight(NamedTuple):
    """int8 weight rows ``q`` [V, d] (row stride a multiple of 16 bytes) and their fp32 scales [V]."""

    q: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def from_weight(cls, weight: torch.Tensor) -> "Int8Weight":
        """Quantises an ``nn.Linear`` weight ``[V, d]``, one scale per vocabulary id."""
        return cls(*quantize_rows(weight))

    def dequantize(self) -> torch.Tensor:
        """The fp32 weight that the int8 rows stand for."""
        return self.q.float() * self.scale[:, None]


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 rows and their fp32 scales: ``scale = max|x| * (1 / 127)`` of each
    row (the reciprocal and the product rounded to fp32) and ``q = round(x /
    scale)`` (half to even), held to -127 .. 127 (only fp32 rows below 2.3e-41,
    whose scales keep a few bits, pass that).  A row of zeros gives zeros and scale
    0; a row with a NaN or an infinity gives zeros and scale NaN.  The int8 rows
    start on 16-byte boundaries (``q`` may be a view of wider rows)."""
    stride = matrix(x, "x")
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x has no columns")
    wide = (cols + 15) // 16 * 16
    q = torch.empty((rows, wide), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    a = N.sized(N.MtrQuantizeArgs, x=x.data_ptr(), x_row_stride=stride, x_dtype=DTYPES[x.dtype], rows=rows, cols=cols,
                q=q.data_ptr(), q_row_stride=wide, scale=scale.data_ptr())
    launch_on(x.device, N.quantize_rows_launch, a)
    return q[:, :cols], scale


def lmhead_i8_args(hidden: torch.Tensor, weight_q: torch.Tensor, weight_scale: torch.Tensor,
                   out: torch.Tensor) -> tuple[N.MtrLmHeadI8Args, torch.Tensor | None]:
    """The launch arguments and the workspace they point to (to be kept until the launch)."""
    hs, ws, ls = matrix(hidden, "hidden"), matrix(weight_q, "weight_q", (torch.int8,)), matrix(out, "logits")
    device = hidden.device
    rows, d = hidden.shape
    vocab = weight_q.shape[0]
    for t, what in ((weight_q, "weight_q"), (weight_scale, "weight_scale"), (out, "logits")):
        same_device(t, device, what)
    if weight_q.shape[1] != d:
        raise ValueError(f"hidden d_model {d} != weight d_model {weight_q.shape[1]}")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (vocab,) or (vocab > 1 and weight_scale.stride(0) != 1):
        raise ValueError(f"weight_scale must be a contiguous float32 vector of {vocab} elements")
    if out.shape[0] != rows or out.shape[1] != vocab:
        raise ValueError("logits must be [hidden rows, vocab]")
    if vocab == 1:
        ws = (d + 15) // 16 * 16
    need = N.lmhead_i8_workspace(rows, d, vocab)  # 0 for few rows
    work = hidden.new_empty(need, dtype=torch.uint8) if need else None
    a = N.sized(N.MtrLmHeadI8Args, hidden=hidden.data_ptr(), hidden_row_stride=hs, weight=weight_q.data_ptr(),
                weight_row_stride=ws, weight_scale=weight_scale.data_ptr(), logits=out.data_ptr(), logits_row_stride=ls,
                hidden_dtype=DTYPES[hidden.dtype], logits_dtype=DTYPES[out.dtype], rows=rows, d_model=d, vocab=vocab,
                workspace=work.data_ptr() if need else None, workspace_bytes=need)
    return a, work


def lm_head_logits_int8(hidden: torch.Tensor, weight_q: torch.Tensor, weight_scale: torch.Tensor,
                        out: torch.Tensor | None = None, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``proj_out(hidden)`` with an int8 weight: ``[R, V]`` logits from hidden
    states ``[R, d]`` (float32, bfloat16 or float16), weight rows ``[V, d]``
    whose row stride is a multiple of 16 bytes (as :func:`quantize_rows` lays
    them out) and their scales ``[V]``.  The logits are ``out``, or a new tensor
    of ``out_dtype``; any of the three dtypes.  Not differentiable.  Logits that a
    wait that gave up left without a value are NaN
    (:func:`~mapperatorinator_b200.sampling.projection_timeouts`)."""
    if out is None:
        if out_dtype not in DTYPES:
            raise TypeError(f"out_dtype {out_dtype} is not supported (float32, bfloat16, float16)")
        out = hidden.new_empty((hidden.shape[0], weight_q.shape[0]), dtype=out_dtype)
    a, work = lmhead_i8_args(hidden, weight_q, weight_scale, out)
    launch_on(hidden.device, N.lmhead_i8_launch, a)
    return out
