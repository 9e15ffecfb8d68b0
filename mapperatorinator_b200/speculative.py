"""Verification of drafted tokens (speculative decoding).

A draft model proposes the next tokens of each sequence, the target scores all of
them in one pass, and ``verify_drafts`` decides in one call which are kept and
what follows them, so that the tokens are distributed as if the target had
written them alone: the counterpart of
:func:`~mapperatorinator_b200.sampling.sample_next_tokens` for several positions
at once.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .int8_head import DTYPES, launch_on, no_tangent, same_device


class Verified(NamedTuple):
    """What :func:`verify_drafts` gives for B sequences of K drafts."""

    tokens: torch.Tensor    # [B, K + 1] int64: accepted drafts, the new token, pad_token_id
    accepted: torch.Tensor  # [B] int32: how many drafts were accepted
    logprobs: torch.Tensor  # [B, K + 1] float32: log p of the tokens (sums of fp32 terms), 0 for padding


def _cube(t: torch.Tensor, what: str) -> tuple[int, int]:
    """Checks a [B, J, V] CUDA tensor with unit last stride; its batch and position strides."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype not in DTYPES:
        raise TypeError(f"{what} dtype {t.dtype} is not supported ({', '.join(str(d)[6:] for d in DTYPES)})")
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{what} must be a [B, positions, V] tensor with unit last stride")
    # the stride of a single row means nothing and may be anything
    pos = t.stride(1) if t.shape[1] > 1 else max(t.shape[2], 1)
    return (t.stride(0) if t.shape[0] > 1 else 0), pos


def _rows(t: torch.Tensor, what: str, dtypes, rows: int, cols: int, device: torch.device) -> int:
    if t.dtype not in dtypes:
        raise TypeError(f"{what} dtype {t.dtype} is not supported ({', '.join(str(d)[6:] for d in dtypes)})")
    if t.shape != (rows, cols) or (cols > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} must be [{rows}, {cols}] with unit column stride")
    same_device(t, device, what)
    return t.stride(0) if rows > 1 else cols


def verify_drafts(target_logits: torch.Tensor, draft_ids: torch.Tensor, draft_logits: torch.Tensor | None = None, *,
                  uniforms: torch.Tensor | None = None, generator: torch.Generator | None = None, temperature: float = 1.0,
                  draft_temperature: float | None = None, do_sample: bool = True, pad_token_id: int = 0,
                  status: torch.Tensor | None = None) -> Verified:
    """Accepts or replaces the drafted tokens of B sequences.

    ``target_logits`` is ``[B, K + 1, V]`` (float32, bfloat16 or float16, any batch
    stride, position stride >= V): the target's logits -- processed scores, if a chain
    applies -- after the prefix and after each draft.  ``draft_ids`` is ``[B, K]``
    int64 or int32, ``draft_logits`` ``[B, K, V]`` of the target's dtype: what the
    drafts were drawn from, or None for drafts without a distribution (looked up,
    or a greedy draft model's).  K is at most 128, and may be 0.

    With ``p = softmax(target / temperature)``, ``q = softmax(draft /
    draft_temperature)`` (default: ``temperature``) and ``uniforms`` ``[B, K + 1]``
    float32 in [0, 1) (default: drawn with ``generator``), draft j is accepted while
    ``uniforms[:, j] q(draft) < p(draft)``.  In the place of the first that is not a
    token is drawn from ``max(p - q, 0)`` by ``uniforms[:, K]``, behind the last one
    from ``p``: the smallest id whose running sum exceeds the uniform's share.  With
    ``do_sample=False`` drafts are accepted while they are the target's first
    maximum, which is also the new token; ``draft_logits`` and ``uniforms`` are not
    read then.

    - A probability of 2^-1000 of the row's largest or less counts as 0: a mask of the
      type's lowest value forbids a token, as -inf does, whatever the uniform.
    - A draft id below 0 ends a sequence's drafts (uneven lengths); so does one >= V,
      which also sets the ``bad_id`` bit.
    - Where the deciding target row holds a NaN or +inf, or only masked scores, the
      new token is ``pad_token_id``; such a draft row refuses its token, and ``p``
      replaces it.  ``status`` (int32 ``[B]``) receives the bits that
      :func:`~mapperatorinator_b200.sampling.row_status_report` reads.
    - A uniform outside [0, 1) is clamped (``bad_uniform``).

    Deterministic, without a host sync, capturable in a CUDA graph when ``uniforms``
    are given.  Not differentiable: ``logprobs`` carry no graph
    (:func:`~mapperatorinator_b200.scoring.token_logprobs` of the tokens does), and
    logits with a forward-mode tangent are refused."""
    no_tangent("verified tokens", target_logits, draft_logits if do_sample else None)
    t_batch, t_pos = _cube(target_logits, "target_logits")
    batch, more, vocab = target_logits.shape
    device, drafts = target_logits.device, more - 1
    if drafts < 0:
        raise ValueError("target_logits must have one position at least")
    ids_stride = _rows(draft_ids, "draft_ids", (torch.int64, torch.int32), batch, drafts, device)
    if draft_temperature is None:
        draft_temperature = temperature
    a = N.sized(N.MtrVerifyArgs, target_logits=target_logits.data_ptr(), target_batch_stride=t_batch, target_pos_stride=t_pos,
                draft_ids=draft_ids.data_ptr() if drafts else None, ids_row_stride=ids_stride,
                logits_dtype=DTYPES[target_logits.dtype], ids_dtype=N.IDS_I32 if draft_ids.dtype == torch.int32 else N.IDS_I64,
                batch=batch, drafts=drafts, vocab=vocab, do_sample=int(bool(do_sample)), temperature=float(temperature),
                draft_temperature=float(draft_temperature), pad_id=int(pad_token_id))
    if do_sample:
        if draft_logits is not None:
            d_batch, d_pos = _cube(draft_logits, "draft_logits")
            if draft_logits.dtype != target_logits.dtype:
                raise TypeError(f"draft_logits dtype {draft_logits.dtype} is not the target's ({target_logits.dtype})")
            if draft_logits.shape != (batch, drafts, vocab):
                raise ValueError(f"draft_logits must be [{batch}, {drafts}, {vocab}]")
            same_device(draft_logits, device, "draft_logits")
            if drafts:
                a.draft_logits, a.draft_batch_stride, a.draft_pos_stride = draft_logits.data_ptr(), d_batch, d_pos
        if uniforms is None:
            uniforms = torch.rand((batch, more), device=device, generator=generator, dtype=torch.float32)
        a.uniforms_row_stride = _rows(uniforms, "uniforms", (torch.float32,), batch, more, device)
        a.uniforms = uniforms.data_ptr()
    if status is not None:
        if status.dtype != torch.int32 or status.shape != (batch,) or not status.is_contiguous():
            raise ValueError(f"status must be a contiguous int32 vector of {batch} elements")
        same_device(status, device, "status")
        a.out_status = status.data_ptr()
    new = target_logits.new_empty
    tokens, accepted = new((batch, more), dtype=torch.int64), new(batch, dtype=torch.int32)
    logprobs = new((batch, more), dtype=torch.float32)
    a.out_tokens, a.out_accepted, a.out_logprobs = tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr()
    need = N.verify_workspace(batch, drafts, vocab, a.logits_dtype)  # 0 for few short rows
    if need:
        work = new(need, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
    launch_on(device, N.verify_launch, a)
    return Verified(tokens, accepted, logprobs)
