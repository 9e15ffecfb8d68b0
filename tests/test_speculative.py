"""Verification of drafted tokens against the definition in float64.

Tokens and counts are whole numbers and have to be equal: the kernels decide in
double what fp32 sums leave open, so only borders within 2^-45 or so of a uniform
could differ, which no input here comes near (uniforms are multiples of 2^-24, and
the closest ones are tested).  Log probabilities: the log-sum-exp is that of fp32
terms or better, within e_S = 2^-22 + 3 2^-24 log V + 16 2^-24 + 36 2^-22 (a term,
its argument, 16 fp32 additions, moves to a larger maximum), then one rounding."""

import ctypes
import math

import numpy as np
import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.speculative import verify_drafts

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LP_TOL = 37 * 2.0 ** -22 + (3 * 12 + 16) * 2.0 ** -24


def softmax(x, t):
    """float64 softmax and log softmax of one row; None where it has none."""
    x = x.double() / t
    if bool(torch.isnan(x).any()) or bool((x == math.inf).any()):
        return "nonfinite"
    if bool((x == -math.inf).all()):
        return "all_masked"
    lp = torch.log_softmax(x, 0)
    return lp.exp(), lp


def draw(w, u):
    run = torch.cumsum(w, 0)
    return int(torch.searchsorted(run, (u * run[-1])[None], right=True))


def reference(target, ids, draft, uniforms, t=1.0, dt=None, do_sample=True, pad=0):
    target, ids = target.cpu(), ids.cpu()
    draft = draft.cpu() if draft is not None else None
    batch, more, vocab = target.shape
    k = more - 1
    tokens = torch.full((batch, more), pad, dtype=torch.int64)
    logprobs = torch.zeros((batch, more), dtype=torch.float64)
    accepted = torch.zeros(batch, dtype=torch.int32)
    status = [set() for _ in range(batch)]
    for b in range(batch):
        u = None
        if do_sample:
            u = uniforms[b].cpu().double()
        at = 0

        def clamped(j):
            v = float(u[j])
            if not 0.0 <= v < 1.0:
                status[b].add("bad_uniform")
                v = 0.0 if not v >= 0.0 else 1.0 - 2.0 ** -24
            return torch.tensor(v, dtype=torch.float64)

        while True:
            token = int(ids[b, at]) if at < k else -1
            if token >= vocab:
                status[b].add("bad_id")
                token = -1
            p = softmax(target[b, at], t)
            if token < 0:
                w = None if isinstance(p, str) else p[0]
                break
            if isinstance(p, str):
                w = None
                break
            if not do_sample:
                if int(target[b, at].float().argmax()) == token:
                    tokens[b, at], logprobs[b, at] = token, p[1][token]
                    at += 1
                    continue
                w = p[0]
                break
            v = clamped(at)
            q = None
            if draft is not None:
                q = softmax(draft[b, at], dt or t)
                if isinstance(q, str):
                    status[b].add(q)
                    w = p[0]
                    break
                q = q[0]
            else:
                q = torch.zeros(vocab, dtype=torch.float64)
                q[token] = 1.0
            if v * q[token] < p[0][token]:
                tokens[b, at], logprobs[b, at] = token, p[1][token]
                at += 1
                continue
            w = (p[0] - q).clamp(min=0)
            if not bool(w.sum() > 0):
                w = p[0]
            break
        accepted[b] = at
        if w is None:
            status[b].add(p)
        else:
            new = draw(w, clamped(k)) if do_sample else int(target[b, at].float().argmax())
            tokens[b, at], logprobs[b, at] = new, p[1][new]
    return tokens, accepted, logprobs, status


def check(target, ids, draft, uniforms, t=1.0, dt=None, do_sample=True, pad=0):
    device = target.device
    status = torch.full((target.shape[0],), -1, dtype=torch.int32, device=device)
    r = verify_drafts(target, ids, draft, uniforms=uniforms, temperature=t, draft_temperature=dt, do_sample=do_sample,
                      pad_token_id=pad, status=status)
    tokens, accepted, logprobs, want_status = reference(target, ids, draft, uniforms, t, dt, do_sample, pad)
    assert torch.equal(r.accepted.cpu(), accepted), (r.accepted.cpu() - accepted).nonzero()
    assert torch.equal(r.tokens.cpu(), tokens), (r.tokens.cpu() != tokens).nonzero()
    err = (r.logprobs.cpu().double() - logprobs).abs()
    assert bool((err <= LP_TOL + 2.0 ** -24 * logprobs.abs()).all()), float(err.max())
    got = [{name for bit, name in S.ROW_STATUS_NAMES.items() if int(s) & bit} for s in status.cpu()]
    assert got == want_status, [(i, a, b) for i, (a, b) in enumerate(zip(got, want_status)) if a != b]
    return r


def inputs(device, batch, drafts, vocab, dtype, seed=0, noise=0.7, masked=0.0):
    g = torch.Generator(device=device).manual_seed(seed)
    target = torch.randn((batch, drafts + 1, vocab), generator=g, device=device) * 2.0
    peaks = torch.randint(0, vocab, (batch, drafts + 1, 4), generator=g, device=device)
    target.scatter_add_(2, peaks, torch.full(peaks.shape, 2.0 + math.log(vocab), device=device))
    if masked:
        out = torch.rand(target.shape, generator=g, device=device) < masked
        out.scatter_(2, peaks[:, :, :1], False)
        target.masked_fill_(out, -math.inf)
    draft = (target[:, :drafts] + noise * torch.randn((batch, drafts, vocab), generator=g, device=device)).to(dtype)
    ids = torch.zeros((batch, drafts), dtype=torch.int64, device=device)
    for j in range(drafts):
        ids[:, j] = torch.multinomial(torch.softmax(draft[:, j].float(), 1), 1, generator=g)[:, 0]
    uniforms = torch.rand((batch, drafts + 1), generator=g, device=device)
    return target.to(dtype), ids, draft, uniforms


# ------------------------------------------------------------------ CPU


def _args(**kw):
    base = dict(target_logits=0x1000000, target_batch_stride=500, target_pos_stride=100, draft_logits=0x2000000, draft_batch_stride=400,
                draft_pos_stride=100, draft_ids=0x3000000, ids_row_stride=4, uniforms=0x3100000, uniforms_row_stride=5,
                logits_dtype=N.DTYPE_BF16, batch=10, drafts=4, vocab=100, do_sample=1, temperature=1.0, draft_temperature=1.0,
                out_tokens=0x4000000, out_accepted=0x4100000, workspace=0x5000000, workspace_bytes=1 << 20)
    return N.sized(N.MtrVerifyArgs, **{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(batch=0, target_logits=None), N.OK), (dict(draft_logits=None), N.OK), (dict(drafts=0, draft_ids=None, draft_logits=None), N.OK),
    (dict(do_sample=0, uniforms=None, draft_logits=None), N.OK), (dict(target_batch_stride=0), N.OK), (dict(ids_row_stride=0), N.OK),
    (dict(batch=-1), N.ERR_BAD_SHAPE), (dict(batch=N.MAX_VERIFY_BATCH + 1), N.ERR_BAD_SHAPE), (dict(drafts=-1), N.ERR_BAD_SHAPE),
    (dict(drafts=N.MAX_DRAFTS + 1), N.ERR_BAD_SHAPE), (dict(vocab=0), N.ERR_BAD_SHAPE), (dict(vocab=N.MAX_VOCAB + 1), N.ERR_BAD_SHAPE),
    (dict(logits_dtype=3), N.ERR_BAD_PARAM), (dict(ids_dtype=2), N.ERR_BAD_PARAM), (dict(do_sample=2), N.ERR_BAD_PARAM),
    (dict(temperature=0.0), N.ERR_BAD_PARAM), (dict(temperature=math.nan), N.ERR_BAD_PARAM), (dict(draft_temperature=-1.0), N.ERR_BAD_PARAM),
    (dict(draft_temperature=math.inf), N.ERR_BAD_PARAM), (dict(temperature=1e-40), N.ERR_BAD_PARAM),
    (dict(target_logits=None), N.ERR_NULL_ARG), (dict(draft_ids=None), N.ERR_NULL_ARG), (dict(uniforms=None), N.ERR_NULL_ARG),
    (dict(out_tokens=None), N.ERR_NULL_ARG), (dict(out_accepted=None), N.ERR_NULL_ARG), (dict(workspace=None, workspace_bytes=0), N.OK),
    (dict(batch=149, workspace=None), N.ERR_NULL_ARG),
    (dict(target_pos_stride=99), N.ERR_BAD_SHAPE), (dict(draft_pos_stride=99), N.ERR_BAD_SHAPE), (dict(target_batch_stride=-1), N.ERR_BAD_SHAPE),
    (dict(batch=149, workspace_bytes=149 * 9 * 16 - 1), N.ERR_BAD_SHAPE), (dict(batch=149, workspace_bytes=149 * 9 * 16), N.OK), (dict(workspace=0x5000008), N.ERR_ALIGNMENT),
    (dict(target_logits=0x1000001), N.ERR_ALIGNMENT), (dict(draft_ids=0x3000004), N.ERR_ALIGNMENT), (dict(uniforms=0x3100002), N.ERR_ALIGNMENT),
    (dict(out_tokens=0x4000004), N.ERR_ALIGNMENT), (dict(out_tokens=0x3000000), N.ERR_BAD_PARAM), (dict(out_tokens=0x3100000), N.ERR_BAD_PARAM),
    (dict(batch=149, out_logprobs=0x5000000), N.ERR_BAD_PARAM), (dict(struct_size=8), N.ERR_ABI), (dict(abi_version=1), N.ERR_ABI)])
def test_arguments_are_checked_on_the_host(kw, code):
    a = _args(**{k: v for k, v in kw.items() if k not in ("struct_size", "abi_version")})
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_verify_validate(ctypes.byref(a)) == code
    if code != N.OK or a.batch == 0:
        assert lib.mtr_verify_launch(ctypes.byref(a), None) == code


@pytest.mark.parametrize("field,need", [("out_tokens", 8 * 149 * 5), ("out_accepted", 4 * 149), ("out_logprobs", 4 * 149 * 5), ("out_status", 4 * 149),
                                        ("workspace", 16 * 149 * 9)])
def test_what_is_written_overlaps_nothing_that_is_read(field, need):
    lib = N.load()
    ok = dict(batch=149, out_logprobs=0x4200000, out_status=0x4300000)

    def code(at, **kw):
        return lib.mtr_verify_validate(ctypes.byref(_args(**{**ok, **kw, field: at})))

    # the last byte of each input, and the first behind it
    target_end = 0x1000000 + 2 * (148 * 500 + 4 * 100 + 100)
    draft_end = 0x2000000 + 2 * (148 * 400 + 3 * 100 + 100)
    ids_end, u_end = 0x3000000 + 8 * 149 * 4, 0x3100000 + 4 * 149 * 5
    up = lambda v: (v + 15) // 16 * 16  # noqa: E731
    for start, end in ((0x1000000, target_end), (0x2000000, draft_end), (0x3000000, ids_end), (0x3100000, u_end)):
        inside = (end - 1) // 16 * 16
        assert code(start) == N.ERR_BAD_PARAM and code(inside) == N.ERR_BAD_PARAM and code(start - up(need) + 16) == N.ERR_BAD_PARAM
        assert code(up(end)) == N.OK and code(start - up(need)) == N.OK
    # not read: the draft's logits and the uniforms of a greedy call, no draft's
    assert code(0x2000000, do_sample=0) == N.OK and code(0x3100000, do_sample=0) == N.OK and code(0x2000000, draft_logits=None) == N.OK
    # between rows and between positions
    far = dict(target_logits=0x40000000, target_batch_stride=1 << 20, target_pos_stride=1 << 17)
    assert code(0x40000000 + 208, **far) == N.OK and code(0x40000000 + (1 << 18) + 208, **far) == N.OK
    assert code(0x40000000 + (1 << 21) * 3 + (1 << 18) * 2 + 192, **far) == N.ERR_BAD_PARAM
    # one target for all sequences
    assert code(0x1000000 + 992, target_batch_stride=0) == N.ERR_BAD_PARAM and code(0x1000000 + 1008, target_batch_stride=0) == N.OK


def test_workspace_sizes():
    assert N.verify_workspace(0, 4, 100, 0) == 0 and N.verify_workspace(3, -1, 100, 0) == 0
    assert N.verify_workspace(64, 4, 4096, N.DTYPE_BF16) == 0             # one launch for all
    assert N.verify_workspace(64, 8, 8192, N.DTYPE_BF16) == 64 * 17 * 16  # a run a row
    assert N.verify_workspace(1, 0, 131072, N.DTYPE_F32) == 16 * 16      # 16 runs
    assert N.verify_workspace(N.MAX_VERIFY_BATCH, N.MAX_DRAFTS, 131072, 0) == (257 << 20) * 16


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        verify_drafts(torch.zeros((2, 3, 16)), torch.zeros((2, 2), dtype=torch.int64))


def test_the_definition_draws_from_the_target():
    """Whatever the draft, the first token is distributed as the target: over all uniforms on a grid."""
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn((1, 2, 5), generator=g), torch.randn((1, 1, 5), generator=g)
    q = torch.softmax(y[0, 0].double(), 0)
    seen = torch.zeros(5, dtype=torch.float64)
    n = 64
    for draft in range(5):
        for i in range(n):
            for j in range(n):
                u = torch.tensor([[(i + 0.5) / n, (j + 0.5) / n]])
                first = reference(x, torch.tensor([[draft]]), y, u)[0][0, 0]
                seen[first] += float(q[draft]) / (n * n)
    # each of the 10 borders moves less than one cell of a grid line
    assert float((seen - torch.softmax(x[0, 0].double(), 0)).abs().max()) < 10 / n


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 0, 1), (1, 1, 1), (2, 1, 2), (3, 2, 7), (1, 4, 4096), (64, 4, 4096), (7, 8, 4099), (200, 3, 513), (5, 40, 300),
                                                (2, 128, 40), (6, 2, 65533), (1, 5, 131072), (3, 1, 16384), (150, 1, 9001)])
def test_drafts_with_a_distribution(cuda_device, dtype, batch, drafts, vocab):
    check(*inputs(cuda_device, batch, drafts, vocab, dtype, seed=batch + vocab))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 1, 2), (64, 8, 4096), (9, 3, 5001), (2, 6, 131072), (33, 33, 100)])
def test_drafts_without_a_distribution_and_uneven(cuda_device, dtype, batch, drafts, vocab):
    target, ids, _, u = inputs(cuda_device, batch, drafts, vocab, dtype, seed=drafts, masked=0.3)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    length = torch.randint(0, drafts + 1, (batch, 1), generator=g, device=cuda_device)
    ids = ids.masked_fill(torch.arange(drafts, device=cuda_device) >= length, -1)
    check(target, ids.int(), None, u, 0.8, pad=-7)
    check(target, ids, None, u * 0.01)  # mostly accepted


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 0, 1), (1, 4, 4096), (64, 6, 4099), (3, 2, 131072), (20, 40, 50), (5, 3, 9)])
def test_greedy(cuda_device, dtype, batch, drafts, vocab):
    target, ids, draft, _ = inputs(cuda_device, batch, drafts, vocab, dtype, seed=vocab)
    if drafts:
        g = torch.Generator(device=cuda_device).manual_seed(2)
        right = torch.rand(ids.shape, generator=g, device=cuda_device) < 0.9
        ids = torch.where(right, target[:, :drafts].float().argmax(2), ids)
    check(target, ids, None, None, 0.7, do_sample=False)
    check(torch.round(target.float() / 4).to(dtype), ids, None, None, do_sample=False)  # many equal maxima
    flat = torch.zeros_like(target)
    flat[..., vocab // 2:] = -0.0
    check(flat, ids * 0, None, None, do_sample=False)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,dt", [(0.05, 0.1), (0.7, None), (1.3, 0.9), (2.0 ** 100, 1.0)])
def test_temperatures(cuda_device, dtype, t, dt):
    target, ids, draft, u = inputs(cuda_device, 40, 4, 700, dtype, seed=11, masked=0.2)
    check(target, ids, draft, u, t, dt)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [50, 4096, 70001])
def test_uniforms_next_to_the_borders(cuda_device, dtype, vocab):
    """Each uniform is the float32 next below or above the border that decides: p / q of a draft, the running sum of a token."""
    batch, drafts = 24, 4
    target, ids, draft, u = inputs(cuda_device, batch, drafts, vocab, dtype, seed=vocab, noise=0.3)
    u = u.cpu()
    side = np.random.default_rng(4)
    t, d, i = target.cpu(), draft.cpu(), ids.cpu()
    for b in range(batch):
        for j in range(drafts + 1):
            p = softmax(t[b, j], 1.0)[0]
            if j < drafts:
                q = softmax(d[b, j], 1.0)[0]
                border = float(p[i[b, j]] / q[i[b, j]])
                if border < 1:
                    low = np.float32(border) if np.float64(np.float32(border)) < border else np.nextafter(np.float32(border), np.float32(0))
                    # mostly accepted, so that later positions come into play
                    u[b, j] = float(low if side.random() < 0.8 else np.nextafter(low, np.float32(1)))
                    continue
                u[b, j] = 0.5
        _, stop, _, _ = reference(t[b:b + 1], i[b:b + 1], d[b:b + 1], u[b:b + 1])
        a = int(stop)
        p = softmax(t[b, a], 1.0)[0]
        w = (p - softmax(d[b, a], 1.0)[0]).clamp(min=0) if a < drafts else p
        run = torch.cumsum(w, 0) / w.sum()
        at = int(torch.searchsorted(run, torch.tensor(side.random(), dtype=torch.float64)))
        border = float(run[min(at, vocab - 1)])
        near = np.float32(border)
        near = near if near < 1 else np.nextafter(np.float32(1), np.float32(0))
        u[b, drafts] = float(near if side.random() < 0.5 else np.nextafter(near, np.float32(0)))
    check(target, ids, draft, u.to(cuda_device))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("noise", [1e-3, 0.05])
@pytest.mark.parametrize("batch,vocab", [(2, 131072), (3, 100003), (40, 20000), (80, 5000)])
def test_distributions_nearly_alike(cuda_device, dtype, noise, batch, vocab):
    """Refused drafts where p and q are next to each other at many ids, or at nearly all of them."""
    target, ids, _, u = inputs(cuda_device, batch, 2, vocab, torch.float32, seed=vocab)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    draft = target[:, :2] + noise * torch.randn((batch, 2, vocab), generator=g, device=cuda_device)
    target, draft = target.to(dtype), draft.to(dtype)
    ids[:, 0] = (draft[:, 0].float() - target[:, 0].float()).argmax(1)  # an id that the draft gives too much
    u[:, 0] = 1.0 - 2.0 ** -20
    r = check(target, ids, draft, u)
    assert int((r.accepted == 0).sum()) > batch // 2


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("vocab", [5, 4096, 20001])
def test_odd_rows(cuda_device, dtype, with_draft, vocab):
    target, ids, draft, u = inputs(cuda_device, 16, 3, vocab, dtype, seed=vocab)
    inf = math.inf
    u[:, :3] *= 0.05                       # mostly accepted
    target[0, 0, vocab - 1] = math.nan
    target[1, 1, 0] = inf
    target[2, 0] = -inf
    target[3, 3] = -inf                    # the bonus position
    draft[4, 0, 1] = math.nan
    draft[5, 1] = -inf
    draft[6, 0, ids[6, 0]] = -inf          # drafted although it could not be
    target[7, 0, ids[7, 0]] = -inf         # forbidden by the target
    ids[8, 1] = vocab                      # out of range
    ids[9, 0] = -100
    u[10, 0], u[10, 3] = -0.5, 1.0
    u[11, 0], u[11, 3] = math.nan, 0.0
    u[12] = 0.0
    target[13, :, 1:] = -inf               # one id left
    target[13, :, 0] = 3.0
    draft[14] = target[14, :3]             # the same distributions: always accepted
    u[14] = 1.0 - 2.0 ** -24
    u[15, 0] = 0.9999
    target[15] = torch.finfo(dtype).min    # masked by the type's lowest value
    target[15, :, 2] = 1.0
    check(target, ids, draft if with_draft else None, u, pad=99)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [37, 4095, 33333])
def test_strided_positions_off_any_boundary(cuda_device, dtype, vocab):
    batch, drafts = 6, 3
    target, ids, draft, u = inputs(cuda_device, batch, drafts, vocab, dtype, seed=3)
    wide = torch.full((drafts + 3, batch + 1, vocab + 5), math.nan, dtype=dtype, device=cuda_device)
    a = wide[1:drafts + 2, :batch, 3:3 + vocab].transpose(0, 1)  # positions outermost
    a.copy_(target)
    other = torch.full((batch, 2 * drafts, vocab + 3), math.nan, dtype=dtype, device=cuda_device)
    d = other[:, ::2, 1:1 + vocab]
    d.copy_(draft)
    many = torch.full((batch, drafts + 4), -1, dtype=torch.int64, device=cuda_device)
    many[:, 2:2 + drafts] = ids
    us = torch.full((batch, drafts + 9), math.nan, device=cuda_device)
    us[:, 5:6 + drafts] = u
    got = check(a, many[:, 2:2 + drafts], d, us[:, 5:6 + drafts])
    plain = verify_drafts(target, ids, draft, uniforms=u)
    assert torch.equal(got.tokens, plain.tokens)
    # one target for all sequences
    check(target[:1].expand(batch, drafts + 1, vocab), ids[:1].expand(batch, drafts), draft[:1].expand(batch, drafts, vocab), u)


@gpu
def test_offsets_that_pass_32_bits(cuda_device):
    """Positions 2^31 elements apart, in one buffer of 2-byte logits."""
    vocab, stride = 1000, 2 ** 30 + 8
    target, ids, draft, u = inputs(cuda_device, 2, 1, vocab, torch.bfloat16, seed=6)
    big = torch.empty(3 * stride + vocab, dtype=torch.bfloat16, device=cuda_device)
    t = big.as_strided((2, 2, vocab), (2 * stride, stride, 1))
    t.copy_(target)
    check(t, ids, draft, u)


@gpu
def test_distribution_of_the_tokens(cuda_device):
    """The first token follows the target's distribution whatever the draft proposes (chi squared, 15 degrees, p = 1e-6: 56.5)."""
    vocab, n = 16, 1 << 18
    g = torch.Generator(device=cuda_device).manual_seed(12)
    target = torch.randn((1, 2, vocab), generator=g, device=cuda_device)
    draft = torch.randn((1, 1, vocab), generator=g, device=cuda_device)
    ids = torch.multinomial(torch.softmax(draft[0, 0], 0), n, replacement=True, generator=g)[:, None]
    r = verify_drafts(target.expand(n, 2, vocab), ids, draft.expand(n, 1, vocab), generator=g)
    count = torch.bincount(r.tokens[:, 0], minlength=vocab).double()
    want = torch.softmax(target[0, 0].double(), 0) * n
    assert float(((count - want) ** 2 / want).sum()) < 56.5
    second = r.tokens[r.accepted == 1, 1]
    want = torch.softmax(target[0, 1].double(), 0) * second.numel()
    count = torch.bincount(second, minlength=vocab).double()
    assert float(((count - want) ** 2 / want).sum()) < 56.5
    assert bool((r.tokens[r.accepted == 0, 1] == 0).all())


@gpu
def test_refusals(cuda_device):
    target, ids, draft, u = inputs(cuda_device, 4, 2, 30, torch.float32)
    for bad in (target.double(), target[0], target.cpu(), target.transpose(1, 2)):
        with pytest.raises((ValueError, TypeError)):
            verify_drafts(bad, ids, draft, uniforms=u)
    for bad in (ids.float(), ids[:3], ids[:, :1], ids.cpu(), ids.t().contiguous().t()):
        with pytest.raises((ValueError, TypeError)):
            verify_drafts(target, bad, draft, uniforms=u)
    for bad in (draft.half(), draft[:, :1], draft[:3], draft.cpu(), draft[:, :, :29]):
        with pytest.raises((ValueError, TypeError)):
            verify_drafts(target, ids, bad, uniforms=u)
    for bad in (u.double(), u[:, :2], u.cpu(), u.t().contiguous().t()):
        with pytest.raises((ValueError, TypeError)):
            verify_drafts(target, ids, draft, uniforms=bad)
    for kw in (dict(temperature=0.0), dict(draft_temperature=-1.0), dict(temperature=math.nan), dict(status=torch.zeros(4, device=cuda_device))):
        with pytest.raises(ValueError):
            verify_drafts(target, ids, draft, uniforms=u, **kw)
    with pytest.raises(ValueError):
        verify_drafts(target[:, :0], ids[:, :0], uniforms=u[:, :0])
    many = torch.zeros((1, N.MAX_DRAFTS + 2, 3), device=cuda_device)
    with pytest.raises(ValueError):
        verify_drafts(many, torch.zeros((1, N.MAX_DRAFTS + 1), dtype=torch.int64, device=cuda_device), do_sample=False)


@gpu
def test_derivatives(cuda_device):
    import torch.autograd.forward_ad as fa

    target, ids, draft, u = inputs(cuda_device, 4, 2, 30, torch.float32)
    with fa.dual_level():
        for t, d in ((fa.make_dual(target, torch.ones_like(target)), draft), (target, fa.make_dual(draft, torch.ones_like(draft)))):
            with pytest.raises(NotImplementedError):
                verify_drafts(t, ids, d, uniforms=u)
        verify_drafts(target, ids, draft, uniforms=u)
    r = verify_drafts(target.clone().requires_grad_(True), ids, draft, uniforms=u)
    assert not r.logprobs.requires_grad


@gpu
def test_no_sequences_and_generated_uniforms(cuda_device):
    target, ids, draft, u = inputs(cuda_device, 4, 2, 30, torch.float32)
    r = verify_drafts(target[:0], ids[:0], draft[:0], uniforms=u[:0])
    assert r.tokens.shape == (0, 3) and r.accepted.shape == (0,)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    a = verify_drafts(target, ids, draft, generator=g)
    g.manual_seed(5)
    b = verify_drafts(target, ids, draft, uniforms=torch.rand((4, 3), device=cuda_device, generator=g))
    assert torch.equal(a.tokens, b.tokens)


@gpu
@pytest.mark.parametrize("batch,vocab", [(3, 50000), (64, 4096)])
def test_same_tokens_on_another_stream_and_in_graphs(cuda_device, batch, vocab):
    sets = [inputs(cuda_device, batch, 4, vocab, torch.bfloat16, seed=s) for s in range(3)]
    want = [verify_drafts(t, i, d, uniforms=u) for t, i, d, u in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = [verify_drafts(t, i, d, uniforms=u) for t, i, d, u in sets]
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    for a, b in zip(want, other):
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.accepted, b.accepted) and torch.equal(a.logprobs, b.logprobs)
    held = [t.clone() for t in sets[0]]
    verify_drafts(held[0], held[1], held[2], uniforms=held[3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = verify_drafts(held[0], held[1], held[2], uniforms=held[3])
    for s, w in zip(sets, want):
        for t, new in zip(held, s):
            t.copy_(new)
        graph.replay()
        assert torch.equal(r.tokens, w.tokens) and torch.equal(r.accepted, w.accepted) and torch.equal(r.logprobs, w.logprobs)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,vocab", [(40, 20001), (2, 131072), (1, 9001), (150, 5000), (64, 4096), (3, 131072), (200, 300)])
@pytest.mark.parametrize("how", ["behind the drafts", "looked up", "refused", "no draft"])
def test_uniform_0_behind_masked_ids(cuda_device, dtype, batch, vocab, how):
    """The smallest id with any weight, although every id of the first half is masked; torch.rand draws 0 too."""
    target, ids, draft, u = inputs(cuda_device, batch, 1, vocab, dtype, seed=vocab)
    first = vocab // 2 + 3
    target[:, :, :first] = -math.inf
    draft[:, :, :first] = -math.inf
    gap = draft[:, 0].float() - target[:, 0].float()
    gap[:, :first] = -math.inf
    ids[:, 0] = gap.argmax(1)  # an id that the draft gives too much
    u[:, 0] = 0.0 if how == "behind the drafts" else 1.0 - 2.0 ** -24
    u[:, 1] = 0.0
    u[::3, 1] = -1.0
    if how == "no draft":
        ids[:] = -1
    r = check(target, ids, None if how == "looked up" else draft, u, pad=-7)
    assert bool((r.accepted == (1 if how == "behind the drafts" else 0)).all()) or how == "looked up"


@gpu
@pytest.mark.parametrize("batch,vocab", [(40, 20001), (2, 131072), (64, 4096), (200, 300)])
@pytest.mark.parametrize("below", [600.0, 630.0, 650.0, 680.0])
def test_uniform_0_and_weights_next_to_nothing(cuda_device, batch, vocab, below):
    """Ids of probability e^-600 and less behind masked ones: with a uniform of 0 the border is within double's rounding of
    many ids, but the token is one that has some weight."""
    target, ids, _, u = inputs(cuda_device, batch, 1, vocab, torch.float32, seed=vocab)
    a, z = vocab // 4, vocab // 2
    target[:, :, :a] = -math.inf
    target[:, :, a:z] = -below
    u[:, 1] = 0.0
    status = torch.full((batch,), -1, dtype=torch.int32, device=cuda_device)
    r = verify_drafts(target, torch.full_like(ids, -1), None, uniforms=u, pad_token_id=-7, status=status)
    assert bool((r.tokens[:, 0] >= a).all()) and bool((r.tokens[:, 0] <= z + target[:, 0, z:].isfinite().float().argmax(1)).all())
    assert bool((status == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,vocab", [(1, 7), (40, 4096), (200, 1000), (8, 4099), (80, 4099), (3, 131072), (80, 20001), (1, 65533)])
def test_a_draft_that_is_the_target_and_could_not_be_drafted(cuda_device, dtype, batch, vocab):
    """p - q is 0 everywhere, and the token comes from p."""
    target, ids, _, u = inputs(cuda_device, batch, 2, vocab, dtype, seed=vocab)
    ids[:, 0] = torch.arange(batch, device=cuda_device) % vocab
    target[:, 0].scatter_(1, ids[:, :1], -math.inf)
    u[:, 2] = (torch.arange(batch, device=cuda_device) + 0.37) / batch
    r = check(target, ids, target[:, :2].clone(), u)
    assert bool((r.accepted == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,batch", [(300, 200), (513, 96), (1000, 96), (4096, 96), (4096, 8), (20001, 80), (131072, 24), (131072, 2)])
def test_uniforms_on_the_borders_of_equal_ids(cuda_device, dtype, vocab, batch):
    """n equally probable ids between masked ones and u = j / 16 with u n whole: the border lies on the running sum of
    u n ids, so rounding decides between two neighbours, and a masked id or none is neither."""
    g = torch.Generator(device=cuda_device).manual_seed(vocab)
    keep = torch.rand((batch, vocab), generator=g, device=cuda_device) < 0.3 + 0.4 * torch.rand((batch, 1), generator=g, device=cuda_device)
    rank = torch.cumsum(keep, 1)
    keep &= rank <= rank[:, -1:] // 16 * 16
    n = keep.sum(1)
    rank = torch.cumsum(keep, 1) - 1  # of an id among those that are left
    target = torch.where(keep, 0.25, -math.inf)[:, None].to(dtype)
    none = torch.empty((batch, 0), dtype=torch.int64, device=cuda_device)
    for j in range(16):
        u = torch.full((batch, 1), j / 16, device=cuda_device)
        token = verify_drafts(target, none, uniforms=u, pad_token_id=-7).tokens
        assert bool((token >= 0).all())
        assert bool(keep.gather(1, token).all())
        off = rank.gather(1, token)[:, 0] - n * j // 16
        assert bool(((off == 0) | (off == -1)).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 4096, 20001])
@pytest.mark.parametrize("how", ["with a draft", "a draft that is masked too", "looked up"])
def test_masks_of_the_lowest_value_forbid(cuda_device, dtype, vocab, how):
    """A drafted token that the target masks by its type's lowest value is refused whatever the uniform, 0 among them
    (e^-65504 is not 0, but no token of such a probability is ever wanted), and is not drawn either."""
    batch = 64
    target, ids, draft, u = inputs(cuda_device, batch, 1, vocab, dtype, seed=vocab)
    low = torch.finfo(dtype).min
    target[:, :, : vocab // 2] = low
    ids[:, 0] = torch.arange(batch, device=cuda_device) % (vocab // 2)
    if how == "a draft that is masked too":
        draft[:, :, : vocab // 2] = low
    u[: batch // 2, 0] = 0.0
    u[::4, 1] = 0.0
    r = check(target, ids, None if how == "looked up" else draft, u, pad=-7)
    assert bool((r.accepted == 0).all()) and bool((r.tokens[:, 0] >= vocab // 2).all())


@gpu
@pytest.mark.parametrize("stateful", [False, True])
def test_scores_of_the_processor_chain(cuda_device, stateful):
    """Drafting and verifying through the framework's chain, position by position: every token is one that the chain allows
    behind what precedes it, and a stateful chain gives the scores of a fresh one."""
    from mapperatorinator_b200.logit_processors import FusedLogitsProcessor

    batch, drafts, vocab, shifts = 8, 3, 600, (10, 410)
    make = lambda state: FusedLogitsProcessor(vocab_size=vocab, time_shift_range=shifts, sos_ids=(1,), stateful_monotonic=state,  # noqa: E731
                                              temperature=0.8, top_k=40, top_p=0.95)
    target_chain, draft_chain = make(stateful), make(stateful)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    table = torch.randn((vocab, vocab), generator=g, device=cuda_device) * 2  # a model of the last token
    other = table + 0.5 * torch.randn((vocab, vocab), generator=g, device=cuda_device)
    history = torch.randint(10, 100, (batch, 4), generator=g, device=cuda_device)
    history[:, 0] = 1
    for _ in range(4):
        seen, drafted, q = history, [], []
        for _ in range(drafts):
            q.append(draft_chain(seen, other[seen[:, -1]].clone()).clone())
            drafted.append(torch.multinomial(torch.softmax(q[-1], 1), 1, generator=g))
            seen = torch.cat([seen, drafted[-1]], 1)
        ids, q = torch.cat(drafted, 1), torch.stack(q, 1)
        scores, fresh = [], []
        for j in range(drafts + 1):
            before = torch.cat([history, ids[:, :j]], 1)
            scores.append(target_chain(before, table[before[:, -1]].clone()).clone())
            fresh.append(make(False)(before, table[before[:, -1]].clone()).clone())
        scores = torch.stack(scores, 1)
        assert torch.equal(scores, torch.stack(fresh, 1))
        r = check(scores, ids, q, torch.rand((batch, drafts + 1), generator=g, device=cuda_device))
        for b in range(batch):
            for j in range(int(r.accepted[b]) + 1):
                assert bool(scores[b, j, r.tokens[b, j]] > -math.inf)
        # the shortest run of new tokens, so that the histories stay one tensor
        history = torch.cat([history, r.tokens[:, : int(r.accepted.min()) + 1]], 1)
