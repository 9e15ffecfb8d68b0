"""Distillation losses and their gradient against the formulas in float64, and
the gradient against differences.

Tolerances.  With S the teacher's ids and d_v = (logit_v - max outside S) / T, the
sum outside S, R = sum e^(d_v), is of fp32 terms: ex2.approx is within 2^-22
relative, its argument within 3 * 2^-24 |d| of d; a thread adds at most 16 pairs in
fp32 and the rest in double; a sum is moved to a larger maximum at most 20 times
(16 tiles and the joins), each within 2^-22.  So R is within
    e_R = 21 2^-22 + 16 2^-24 + 3 2^-24 mean |d|
relative.  What belongs to S is computed in double.  Of log S = log(in + rest) a
share q_t comes from R, so
    |loss error| <= max(q_t, p_t) e_R + 2^-24 |loss| + 2^-40 (1 + sum p |log q|).
A gradient inside S is (q_v (P + p_t) - p_v) g / T in double, q_v within q_t e_R and
2^-40; outside it is e^(d_v) times one number of the row, made of two parts whose
magnitudes add to B = q_v P + p_t (1 - q_t) q_v / q_t: within
    B (2 e_R + 2^-22 + 3 2^-24 |d| + 2^-23) + eps / 2 |value|
and the smallest subnormal; e^(d_v) below 2^-126 counts as 0."""

import ctypes
import math

import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.distillation import distillation_loss, distillation_loss_and_grad
from mapperatorinator_b200.scoring import token_logprobs

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def reference(logits, ids, lps, tail, temperature, g=None):
    """The definition in float64; the losses, the gradient and the bounds of both."""
    x = logits.detach().double() / temperature
    rows, vocab = x.shape
    ids, l = ids.long(), lps.double()
    valid = (ids >= 0) & (ids < vocab)
    bad = (torch.isnan(x) | (x == math.inf)).any(1) | (valid & ~(l < math.inf)).any(1)
    none = (x == -math.inf).all(1)
    l = torch.where(valid, l, -math.inf)
    empty = ~valid.any(1)
    if not tail:
        empty |= ~bad & (l == -math.inf).all(1)
    odd = bad | empty | none
    x = torch.where(odd[:, None], 0.0, x)  # computed, not used
    if not tail:
        l = torch.where(odd[:, None], -1.0, l)
        l = l - torch.logsumexp(l, 1, keepdim=True)
    p = torch.exp(torch.where(bad[:, None], -math.inf, l))
    p = torch.where(valid, p, 0.0)
    mass = p.sum(1)
    p_t = 1.0 - mass if tail else torch.zeros_like(mass)
    p_t = torch.where(p_t < 2.0 ** -20, 0.0, p_t)
    inside = torch.zeros((rows, vocab + 1), dtype=torch.bool, device=x.device)
    inside.scatter_(1, torch.where(valid, ids, vocab), True)
    inside = inside[:, :vocab]
    listed = torch.zeros((rows, vocab + 1), dtype=torch.float64, device=x.device)
    listed.scatter_add_(1, torch.where(valid, ids, vocab), p)
    listed = listed[:, :vocab]
    logq = x - torch.logsumexp(x, 1, keepdim=True)
    q = torch.exp(logq)
    outer = torch.where(inside, -math.inf, logq)
    top = outer.amax(1)
    top = torch.where(torch.isinf(top), 0.0, top)
    d = outer - top[:, None]  # a row's far logits would swallow the logarithm of their number
    log_rest = torch.logsumexp(d, 1)
    log_qt = top + log_rest
    q_t = torch.exp(log_qt)
    at = torch.where(valid, ids, 0)
    part = torch.where(p > 0, p * (l - logq.gather(1, at)), 0.0)
    loss = part.sum(1) + torch.where(p_t > 0, p_t * (torch.log(p_t) - log_qt), 0.0)
    loss = torch.where(none, math.inf, loss)
    loss = torch.where(empty, 0.0, torch.where(bad, math.nan, loss))
    # bounds
    share = torch.where(torch.isinf(outer), 0.0, torch.exp(d - torch.where(torch.isinf(log_rest), 0.0, log_rest)[:, None]))
    d = torch.where(torch.isinf(outer), 0.0, d)
    e_r = 21 * 2.0 ** -22 + 16 * U + 3 * U * (share * d.abs()).sum(1)
    size = (p * torch.where(p > 0, logq.gather(1, at), 0.0).nan_to_num(0, 0, 0).abs()).sum(1)
    loss_tol = torch.maximum(q_t, p_t) * e_r + U * loss.nan_to_num(0, 0, 0).abs() + 2.0 ** -40 * (1 + size)
    loss_tol = torch.where(odd, 0.0, loss_tol)
    if g is None:
        return loss, loss_tol, None, None
    gt = (g.double() / temperature)[:, None]
    ratio = torch.where((p_t > 0)[:, None], (p_t * (1 - q_t))[:, None] * share, 0.0)
    even = q * mass[:, None]
    grad = torch.where(inside, q * (mass + p_t)[:, None] - listed, even - ratio) * gt
    eps = torch.finfo(logits.dtype).eps / 2
    room = torch.where(inside, q * (mass + p_t)[:, None] * (q_t * e_r + 2.0 ** -40)[:, None] + 2.0 ** -40 * listed,
                       (even + ratio) * (2 * e_r[:, None] + 2.0 ** -22 + 3 * U * d.abs() + 2.0 ** -23)) * gt.abs()
    scale = (mass + torch.where(p_t > 0, p_t * torch.exp(-log_qt), 0.0)).nan_to_num(0, 0, 0)[:, None] * gt.abs()
    room = room + (eps + U) * grad.abs() + torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps + scale * 2.0 ** -125
    grad = torch.where((empty | none)[:, None], 0.0, grad)
    grad = torch.where((bad & ~empty)[:, None], math.nan, grad)
    return loss, loss_tol, grad, room


def close(got, want, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    err = (got - want).abs()[ok] - tol.expand_as(want)[ok]
    assert err.numel() == 0 or float(err.max()) <= 0, (what, float(err.max()))


def inputs(device, rows, vocab, n, dtype, seed=0, scale=2.0, temperature=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    base = torch.randn((rows, vocab), generator=g, device=device) * scale
    logits = (base + torch.randn((rows, vocab), generator=g, device=device)).to(dtype)
    teacher = torch.log_softmax(base / temperature, 1)
    take = min(n, vocab)
    lps, ids = torch.topk(teacher, take, 1)
    if take < n:
        ids = torch.cat([ids, ids.new_full((rows, n - take), -1)], 1)
        lps = torch.cat([lps, lps.new_full((rows, n - take), -math.inf)], 1)
    w = torch.randn((rows,), generator=g, device=device)
    return logits, ids, lps, w


def check(logits, ids, lps, tail, temperature=1.0, g=None):
    loss, grad = distillation_loss_and_grad(logits, ids, lps, g, temperature=temperature, tail=tail)
    alone = distillation_loss(logits, ids, lps, temperature=temperature, tail=tail)
    want, tol, want_grad, room = reference(logits, ids, lps, tail, temperature, torch.ones_like(loss) if g is None else g)
    close(loss, want, tol, "loss")
    assert torch.equal(alone.isnan(), loss.isnan()) and torch.equal(alone[~alone.isnan()], loss[~loss.isnan()])
    close(grad, want_grad, room, "grad")
    leaf = logits.detach().clone().requires_grad_(True) if logits.is_contiguous() else logits.detach().requires_grad_(True)
    other = distillation_loss(leaf, ids, lps, temperature=temperature, tail=tail)
    (by_autograd,) = torch.autograd.grad(other, leaf, torch.ones_like(loss) if g is None else g)
    same = by_autograd.isnan() & grad.isnan()
    assert torch.equal(by_autograd[~same], grad[~same])
    return loss, grad


# ------------------------------------------------------------------ CPU


def _args(**kw):
    base = dict(logits=0x1000000, logits_row_stride=100, teacher_ids=0x2000000, ids_row_stride=8, teacher_logprobs=0x3000000,
                logprobs_row_stride=8, logits_dtype=N.DTYPE_BF16, ids_dtype=N.IDS_I64, rows=10, vocab=100, n=8, temperature=1.0,
                out_loss=0x4000000, grad_logits=0x5000000, grad_row_stride=100)
    return N.sized(N.MtrDistillArgs, **{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0, logits=None), N.OK), (dict(grad_logits=None), N.OK), (dict(out_loss=None, stats=0x6000000), N.OK),
    (dict(ids_row_stride=0, logprobs_row_stride=0), N.OK), (dict(tail=1), N.OK), (dict(n=N.MAX_TEACHER_IDS), N.OK),
    (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(rows=N.MAX_SCORE_ROWS + 1), N.ERR_BAD_SHAPE), (dict(vocab=0), N.ERR_BAD_SHAPE),
    (dict(vocab=N.MAX_VOCAB + 1), N.ERR_BAD_SHAPE), (dict(n=0), N.ERR_BAD_PARAM), (dict(n=N.MAX_TEACHER_IDS + 1), N.ERR_BAD_PARAM),
    (dict(logits_dtype=3), N.ERR_BAD_PARAM), (dict(ids_dtype=2), N.ERR_BAD_PARAM), (dict(tail=2), N.ERR_BAD_PARAM),
    (dict(temperature=0.0), N.ERR_BAD_PARAM), (dict(temperature=math.nan), N.ERR_BAD_PARAM), (dict(temperature=1e-39), N.ERR_BAD_PARAM),
    (dict(temperature=2.0 ** 101), N.ERR_BAD_PARAM), (dict(logits=None), N.ERR_NULL_ARG), (dict(teacher_ids=None), N.ERR_NULL_ARG),
    (dict(teacher_logprobs=None), N.ERR_NULL_ARG), (dict(out_loss=None), N.ERR_NULL_ARG),
    (dict(out_loss=None, grad_logits=None, stats=0x6000000), N.ERR_NULL_ARG), (dict(logits_row_stride=99), N.ERR_BAD_SHAPE),
    (dict(grad_row_stride=99), N.ERR_BAD_SHAPE), (dict(ids_row_stride=-1), N.ERR_BAD_SHAPE), (dict(logits=0x1000001), N.ERR_ALIGNMENT),
    (dict(teacher_ids=0x2000004), N.ERR_ALIGNMENT), (dict(teacher_ids=0x2000004, ids_dtype=N.IDS_I32), N.OK),
    (dict(teacher_logprobs=0x3000002), N.ERR_ALIGNMENT), (dict(stats=0x6000008), N.ERR_ALIGNMENT), (dict(out_status=2), N.ERR_ALIGNMENT),
    (dict(grad_logits=0x1000000), N.ERR_BAD_PARAM), (dict(grad_logits=0x1000000 + 9 * 200), N.ERR_BAD_PARAM),
    (dict(grad_logits=0x2000000), N.ERR_BAD_PARAM), (dict(grad_logits=0x3000000), N.ERR_BAD_PARAM),
    (dict(g_loss=0x5000000), N.ERR_BAD_PARAM), (dict(struct_size=8), N.ERR_ABI), (dict(abi_version=1), N.ERR_ABI)])
def test_arguments_are_checked_on_the_host(kw, code):
    a = _args(**{k: v for k, v in kw.items() if k not in ("struct_size", "abi_version")})
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_distill_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_distill_launch(ctypes.byref(a), None) == code


@pytest.mark.parametrize("field,size", [("out_loss", 4), ("stats", 16), ("out_status", 4)])
def test_what_is_written_overlaps_nothing_that_is_read(field, size):
    lib = N.load()
    ok = dict(rows=100, stats=0x7000000, out_status=0x7100000, g_loss=0x6000000)

    def code(at, **kw):
        return lib.mtr_distill_validate(ctypes.byref(_args(**{**ok, **kw, field: at})))

    # the last byte of logits, ids, log probabilities, gradients of the losses, gradient, and the first behind it
    up = lambda v: (v + 15) // 16 * 16  # noqa: E731
    for start, n in ((0x1000000, 100 * 200), (0x2000000, 100 * 64), (0x3000000, 100 * 32), (0x6000000, 400), (0x5000000, 100 * 200)):
        end = start + n
        assert code(start) == N.ERR_BAD_PARAM and code((end - 1) // 16 * 16) == N.ERR_BAD_PARAM
        assert code(start - up(100 * size) + 16) == N.ERR_BAD_PARAM
        assert code(up(end)) == N.OK and code(start - up(100 * size)) == N.OK
    assert code(0x1000000 + 9 * 256 + 208, rows=1, logits_row_stride=128) == N.OK
    assert code(0x2000000 + 64, ids_row_stride=0) == N.OK and code(0x2000000 + 48, ids_row_stride=0) == N.ERR_BAD_PARAM
    # the gradient alone reads the statistics and writes no loss or status
    alone = dict(out_loss=None, stats=0x7000000)
    if field == "stats":
        assert code(0x5000000 + 19792, **alone) == N.ERR_BAD_PARAM and code(0x1000000, **alone) == N.OK
    elif field == "out_status":
        assert code(0x1000000, **alone) == N.OK


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        distillation_loss(torch.zeros((2, 16)), torch.zeros((2, 1), dtype=torch.int64), torch.zeros((2, 1)))


@pytest.mark.parametrize("tail", [False, True])
def test_formula_against_differences(tail):
    g = torch.Generator().manual_seed(3)
    x = torch.randn((4, 13), generator=g, dtype=torch.float64)
    lps, ids = torch.topk(torch.log_softmax(torch.randn((4, 13), generator=g), 1), 5, 1)
    ids[1, 2] = -1
    ids[2, 1] = ids[2, 0]  # an id given twice
    w = torch.randn(4, generator=g)
    _, _, grad, _ = reference(x, ids, lps, tail, 0.7, w)
    h = 1e-5
    for v in range(13):
        step = torch.zeros_like(x)
        step[:, v] = h
        up, down = (reference(x + s, ids, lps, tail, 0.7)[0] for s in (step, -step))
        # third derivatives of a softmax are below 1 / T^3, and sums of 13 doubles keep 1e-15
        assert torch.allclose((up - down) / (2 * h) * w, grad[:, v], atol=1e-9, rtol=0)


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,n", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (7, 40, 40), (64, 4096, 5), (33, 4099, 33), (9, 9001, 128), (300, 513, 32),
                                          (5, 16384, 20), (3, 65533, 64), (2, 131072, 100)])
def test_losses_and_gradients(cuda_device, dtype, tail, rows, vocab, n):
    logits, ids, lps, w = inputs(cuda_device, rows, vocab, n, dtype, seed=rows + vocab)
    check(logits, ids, lps, tail, 1.0, w)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [0.05, 0.7, 3.0, 2.0 ** 100])
def test_temperatures(cuda_device, dtype, tail, temperature):
    logits, ids, lps, w = inputs(cuda_device, 20, 1000, 12, dtype, seed=5, temperature=max(0.3, min(temperature, 5.0)))
    check(logits, ids.int(), lps, tail, temperature, w)


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_logits_serve_as_well_where_the_ids_are_renormalised(cuda_device, tail):
    logits, ids, lps, w = inputs(cuda_device, 30, 500, 7, torch.float32, seed=8)
    if tail:
        check(logits, ids, lps - 0.25, tail, 1.0, w)  # part of the mass outside
    else:
        check(logits, ids, lps + 31.0, tail, 1.0, w)
        check(logits, ids, lps - 200.0, tail, 1.0, w)


def _odd_rows(device, vocab, n, dtype):
    logits, ids, lps, w = inputs(device, 16, vocab, n, dtype, seed=vocab, scale=3.0)
    inf = math.inf
    logits[0] = -inf                                    # all masked
    logits[1, 0] = math.nan
    logits[2, vocab - 1] = inf
    logits[3] = -inf
    logits[3, ids[3, 0]] = 1.0                          # one id left, a teacher's
    logits[4, ids[4, 0]] = -inf                         # the student has no mass where the teacher has some
    ids[5] = -1                                         # no entries
    ids[6, : n // 2 + 1] = -100
    ids[7, 0] = vocab                                   # out of range
    lps[8, 0] = math.nan
    lps[9, n - 1] = inf
    lps[10] = -inf
    ids[11] = -1
    logits[11, 0] = math.nan                            # no entries, whatever the logits hold
    logits[12] = torch.finfo(dtype).min                 # masked by the type's lowest value
    logits[12, ids[12, 0]] = 0.0
    lps[13, : n // 2] = -inf
    logits[14] = 0.0
    if vocab > n:
        keep = torch.zeros(vocab, dtype=torch.bool, device=device)
        keep[ids[15]] = True
        logits[15, ~keep] = -inf                        # no mass outside the ids
    return logits, ids, lps, w


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab,n", [(3, 2), (40, 6), (4096, 20), (5001, 40), (40000, 32)])
def test_rows_that_masks_and_values_make_odd(cuda_device, dtype, tail, vocab, n):
    logits, ids, lps, w = _odd_rows(cuda_device, vocab, n, dtype)
    check(logits, ids, lps, tail, 1.0, w)
    status = torch.full((16,), -1, dtype=torch.int32, device=cuda_device)
    distillation_loss(logits, ids, lps, tail=tail, status=status)
    rep = S.row_status_report(status)
    assert rep["bad_id"] == [7] and rep["all_masked"] == [0]
    assert rep["nonfinite"] == [1, 2, 8, 9]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [3, 40])
def test_entries_without_probability_whatever_the_logits_hold(cuda_device, dtype, n):
    logits, ids, lps, w = inputs(cuda_device, 4, 500, n, dtype)
    lps[:3] = -math.inf
    logits[0, ids[0, 1]] = math.nan
    logits[1, ids[1, 0]] = math.inf
    logits[2] = math.nan
    loss, grad = distillation_loss_and_grad(logits, ids, lps, w)
    leaf = logits.clone().requires_grad_(True)
    (distillation_loss(leaf, ids, lps) * w).sum().backward()
    for g in (grad, leaf.grad):
        assert torch.equal(g[:3], torch.zeros_like(g[:3])) and g[3].any()
    assert torch.equal(loss[:3], torch.zeros_like(loss[:3])) and loss[3].isfinite()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n", [4, 32, 70])
def test_ids_given_twice(cuda_device, dtype, tail, n):
    logits, ids, lps, w = inputs(cuda_device, 24, 300, n, dtype, seed=n)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    ids = torch.gather(ids, 1, torch.randint(0, n, ids.shape, generator=g, device=cuda_device))  # many equal ones
    ids[0] = ids[0, 0]
    lps = torch.log_softmax(lps, 1) - 0.3
    check(logits, ids, lps, tail, 1.0, w)


@gpu
@pytest.mark.parametrize("tail", [False, True])
def test_confident_students_keep_their_digits(cuda_device, tail):
    """Losses and gradients that are small differences: a student near the teacher, with nearly all mass on one id."""
    rows, vocab, n = 64, 4096, 8
    g = torch.Generator(device=cuda_device).manual_seed(2)
    logits = torch.randn((rows, vocab), generator=g, device=cuda_device)
    lead = torch.randint(0, vocab, (rows,), generator=g, device=cuda_device)
    logits[torch.arange(rows, device=cuda_device), lead] += torch.linspace(10.0, 30.0, rows, device=cuda_device)
    lps, ids = torch.topk(torch.log_softmax(logits + 0.01 * torch.randn(logits.shape, generator=g, device=cuda_device), 1), n, 1)
    check(logits, ids, lps, tail, 1.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride,offset,out_stride,out_offset", [
    (100, 101, 1, 100, 0), (4096, 4099, 3, 4099, 3), (4095, 4095, 5, 4100, 2), (20000, 20003, 7, 20003, 7), (8193, 8193, 1, 8193, 1), (5, 9, 3, 5, 0),
    (66000, 66001, 3, 66001, 1)])
def test_strided_rows_off_any_boundary(cuda_device, dtype, vocab, stride, offset, out_stride, out_offset):
    rows, n = 9, min(20, vocab)
    plain, ids, lps, w = inputs(cuda_device, rows, vocab, n, dtype, seed=vocab)
    flat = torch.full((rows * stride + offset + 64,), math.nan, dtype=dtype, device=cuda_device)
    logits = flat[offset:].as_strided((rows, vocab), (stride, 1))
    logits.copy_(plain)
    given = torch.full((rows * out_stride + out_offset + 64,), 7.0, dtype=dtype, device=cuda_device)
    out = given[out_offset:].as_strided((rows, vocab), (out_stride, 1))
    loss, grad = distillation_loss_and_grad(logits, ids, lps, w, tail=True, out=out)
    assert grad is out
    want, tol, want_grad, room = reference(plain, ids, lps, True, 1.0, w)
    close(loss, want, tol, "loss")
    close(grad, want_grad, room, "grad")
    untouched = torch.ones_like(given, dtype=torch.bool)
    untouched[out_offset:].as_strided((rows, vocab), (out_stride, 1)).fill_(False)
    assert (given[untouched] == 7.0).all()
    wide = torch.full((rows, n + 3), -1, dtype=torch.int64, device=cuda_device)
    wide[:, 1:1 + n] = ids
    again, _ = distillation_loss_and_grad(logits, wide[:, 1:1 + n], lps, w, tail=True)
    assert torch.equal(again, loss)


@gpu
def test_one_teacher_row_for_all_and_no_rows(cuda_device):
    logits, ids, lps, w = inputs(cuda_device, 12, 200, 6, torch.bfloat16, seed=4)
    check(logits, ids[:1].expand(12, 6), lps[:1].expand(12, 6), True, 1.0, w)
    loss, grad = distillation_loss_and_grad(logits[:0], ids[:0], lps[:0])
    assert loss.shape == (0,) and grad.shape == (0, 200)
    leaf = logits.clone().requires_grad_(True)
    distillation_loss(leaf, ids, lps).mean().backward()  # an expanded gradient
    want = distillation_loss_and_grad(logits, ids, lps, torch.full((12,), 1 / 12, device=cuda_device))[1]
    assert torch.equal(leaf.grad, want)


@gpu
@pytest.mark.parametrize("rows,vocab,n,dtype", [(9000, 600, 8, torch.bfloat16), (5000, 4097, 20, torch.float16), (2600, 2100, 40, torch.float32),
                                                (1, 131072, 32, torch.float32), (20, 70001, 5, torch.bfloat16), (700, 33000, 16, torch.bfloat16)])
@pytest.mark.parametrize("tail", [False, True])
def test_many_rows_and_few(cuda_device, tail, rows, vocab, n, dtype):
    """The number of threads and CTAs that share a row goes by both sizes."""
    logits, ids, lps, w = inputs(cuda_device, rows, vocab, n, dtype, seed=rows)
    logits[rows // 2, vocab // 3] = math.nan
    logits[rows - 1, : vocab - 3] = -math.inf
    check(logits, ids, lps, tail, 1.3, w)


@gpu
def test_refusals(cuda_device):
    logits, ids, lps, w = inputs(cuda_device, 6, 50, 4, torch.float32)
    for bad in (ids[:5], ids.float(), ids[:, :0], ids[:, :3], ids.cpu(), ids.t()):
        with pytest.raises((ValueError, TypeError)):
            distillation_loss(logits, bad, lps)
    for bad in (lps.double(), lps[:5], lps.cpu(), lps[:, :2]):
        with pytest.raises((ValueError, TypeError)):
            distillation_loss(logits, ids, bad)
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.inf), dict(status=torch.zeros(6, device=cuda_device)),
               dict(status=torch.zeros(5, dtype=torch.int32, device=cuda_device))):
        with pytest.raises(ValueError):
            distillation_loss(logits, ids, lps, **kw)
    with pytest.raises(TypeError):
        distillation_loss(logits.double(), ids, lps)
    with pytest.raises(ValueError):
        distillation_loss(logits, ids, lps.clone().requires_grad_(True))
    wide = ids.new_zeros((6, N.MAX_TEACHER_IDS + 1))
    with pytest.raises(ValueError):
        distillation_loss(logits, wide, wide.float())
    for bad in (w.double(), w[:5], w.cpu()):
        with pytest.raises(ValueError):
            distillation_loss_and_grad(logits, ids, lps, bad)
    for bad in (logits, logits.to(torch.bfloat16), torch.empty((6, 49), device=cuda_device), torch.empty((50, 6), device=cuda_device).t()):
        with pytest.raises(ValueError):
            distillation_loss_and_grad(logits, ids, lps, w, out=bad)
    leaf = logits.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(distillation_loss(leaf, ids, lps).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)
    import torch.autograd.forward_ad as fa
    with fa.dual_level(), pytest.raises(NotImplementedError):
        distillation_loss(fa.make_dual(logits, torch.ones_like(logits)), ids, lps)


@gpu
def test_same_bits_again_on_another_stream_and_in_graphs(cuda_device):
    sets = [inputs(cuda_device, 700, 4099, 20, torch.bfloat16, seed=s) for s in range(3)]
    want = [distillation_loss_and_grad(*s, tail=True) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = [distillation_loss_and_grad(*s, tail=True) for s in sets]
    torch.cuda.current_stream(cuda_device).wait_stream(side)
    for a, b in zip(want, other):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    held = [t.clone() for t in sets[0]]
    out = torch.empty_like(held[0])
    distillation_loss_and_grad(*held, tail=True, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = distillation_loss_and_grad(*held, tail=True, out=out)
    for s, (l, g) in zip(sets, want):
        for t, new in zip(held, s):
            t.copy_(new)
        graph.replay()
        assert torch.equal(loss, l) and torch.equal(out, g)


@gpu
def test_what_scoring_reports_is_what_is_learned(cuda_device):
    """A teacher's alternatives train a student to its distribution: at the teacher's own logits loss and gradient vanish."""
    g = torch.Generator(device=cuda_device).manual_seed(9)
    teacher = torch.randn((50, 700), generator=g, device=cuda_device) * 2
    r = token_logprobs(teacher, top_n=32, temperature=1.5)
    loss, grad = check(teacher, r.top_ids, r.top_logprobs, True, 1.5)
    # the alternatives are fp32 logarithms of about 5: p within 8 2^-24, 33 of them
    assert float(loss.abs().max()) < 1e-5 and float(grad.abs().max()) < 1e-5
    few = token_logprobs(torch.full_like(teacher, -math.inf).scatter_(1, r.top_ids[:, :3], 1.0), top_n=8)
    assert (few.top_ids[:, 3:] == -1).all()
    check(teacher, few.top_ids, few.top_logprobs, True)


@gpu
@pytest.mark.parametrize("order", ["rising", "falling", "as drawn"])
@pytest.mark.parametrize("tail", [False, True])
def test_long_rows_whose_maximum_moves(cuda_device, tail, order):
    """256 threads on rows of 131072 fp32 logits: a thread has 32 tiles of 16, so its sum moves to a larger maximum at most
    31 times, then to its single logit's, the warp's and the row's: e_R = 35 2^-22 + 16 2^-24 + 3 2^-24 mean |d|, 14 2^-22 more
    than where rows are shorter or have 512 threads."""
    rows, vocab, n = 300, 131072, 20
    logits, ids, lps, w = inputs(cuda_device, rows, vocab, n, torch.float32, seed=1)
    if order != "as drawn":
        logits = logits.sort(1, descending=order == "falling").values
    loss, grad = distillation_loss_and_grad(logits, ids, lps, w, tail=tail)
    more = 14 * 2.0 ** -22
    for r in range(0, rows, 60):  # the reference needs some 40 bytes a logit
        part = slice(r, r + 60)
        want, tol, want_grad, room = reference(logits[part], ids[part], lps[part], tail, 1.0, w[part])
        close(loss[part], want, tol + more, "loss")
        # outside the ids room is at least 2 21 2^-22 of the parts' magnitudes, inside the ids q_t 21 2^-22 of one
        close(grad[part], want_grad, room * (1 + 14 / 21), "grad")
