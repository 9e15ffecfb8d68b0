"""Log probabilities of given tokens, entropy, log-sum-exp, top alternatives and
their gradient against the formulas in float64 (and the gradient against
differences).

Tolerances (float32 outputs), with d_v = (logit_v - max) / T and p the
probabilities: ex2.approx is within 2^-22 relative, its argument within
3 * 2^-24 |d| of d (a difference, a product, the rounded factor), and a chain of
c fp32 additions adds c 2^-24 relative.  So log S is within
    e_S = 2^-22 + 3 2^-24 sum p |d| + (V / 256 + 64) 2^-24 + 2^-22 |log S|,
(the last for log1p), a log probability within e_S + 4 2^-24 |log p|, the
log-sum-exp within e_S + 2 2^-24 |lse|, and the entropy, log S plus the mean of
|d|, within e_S + (2^-21 + 3 2^-24 max|d where p counts| + (V / 256 + 64) 2^-23) sum p |d|.
A gradient p (a + b (log p + H)) has relative error e_p = 2^-22 + (3 |d| + 2 |log S|) 2^-24 + e_S
in p, e_H + e_log p in the bracket, and a rounding to its type (eps / 2)."""

import math

import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.scoring import TokenLogprobs, token_logprobs, token_logprobs_backward

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24


def reference(logits, tokens, top_n, temperature=1.0):
    """The definition in float64, row by row semantics included."""
    x = logits.detach().double() / temperature
    rows, vocab = x.shape
    bad = (torch.isnan(x) | (x == math.inf)).any(1)
    none = (x == -math.inf).all(1) & ~bad
    m = torch.where(bad | none, 0.0, x.amax(1).nan_to_num(0.0, 0.0, 0.0))
    d = x - m[:, None]
    p = torch.exp(d)
    s = p.sum(1)
    log_s = torch.log(s)
    logp = d - log_s[:, None]
    p = p / s[:, None]
    ent = -torch.where(p > 0, p * logp, 0.0).sum(1)
    lse = m + log_s
    out = {"d": d, "p": p, "logp": logp, "log_s": log_s, "bad": bad, "none": none}
    nan = torch.full_like(ent, math.nan)
    out["entropy"] = torch.where(bad, nan, torch.where(none, 0.0, ent))
    out["lse"] = torch.where(bad, nan, torch.where(none, -math.inf, lse))
    if tokens is not None:
        has = (tokens >= 0) & (tokens < vocab)
        t = logp.gather(1, torch.where(has, tokens, 0).long()[:, None])[:, 0]
        t = torch.where(bad, nan, torch.where(none, -math.inf, t))
        out["logprobs"] = torch.where(has, t, 0.0)
        out["has"] = has
    raw = logits.detach().double()
    order = torch.argsort(torch.where(bad[:, None], 0.0, -raw), dim=1, stable=True)[:, :top_n]
    ok = (raw.gather(1, order) > -math.inf) & ~bad[:, None]
    ids = torch.where(ok, order, -1)
    lp = torch.where(ok, logp.gather(1, order), -math.inf)
    lp = torch.where(bad[:, None], math.nan, lp)
    if top_n > vocab:
        ids = torch.cat([ids, ids.new_full((rows, top_n - vocab), -1)], 1)
        fill = torch.where(bad, math.nan, -math.inf)[:, None].expand(rows, top_n - vocab)
        lp = torch.cat([lp, fill], 1)
    out["top_ids"], out["top_logprobs"] = ids, lp
    return out


def bounds(ref, vocab):
    d = torch.where(ref["p"] > 0, ref["d"].abs(), 0.0)
    mean = (ref["p"] * d).sum(1)
    chain = vocab / 256 + 64
    es = 2.0 ** -22 * (1 + ref["log_s"].abs()) + 3 * U * mean + chain * U
    eh = es + (2.0 ** -21 + 3 * U * 110 + 2 * chain * U) * mean
    plain = ~(ref["bad"] | ref["none"])  # the other rows are defined to the bit
    return torch.where(plain, es, 0.0), torch.where(plain, eh, 0.0)


def close(got, want, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = torch.isfinite(want)
    err = (got - want).abs()[ok] - tol.expand_as(want)[ok]
    assert err.numel() == 0 or float(err.max()) <= 0, (what, float(err.max()))


def check_forward(r, logits, tokens, top_n, temperature=1.0):
    ref = reference(logits, tokens, top_n, temperature)
    es, eh = bounds(ref, logits.shape[1])
    if tokens is None:
        assert r.logprobs is None
    else:
        close(r.logprobs, ref["logprobs"], es + 4 * U * ref["logprobs"].abs().nan_to_num(0, 0, 0), "logprobs")
    close(r.entropy, ref["entropy"], eh, "entropy")
    close(r.lse, ref["lse"], es + 2 * U * ref["lse"].abs().nan_to_num(0, 0, 0), "lse")
    assert torch.equal(r.top_ids, ref["top_ids"]), "top_ids"
    close(r.top_logprobs, ref["top_logprobs"], es[:, None] + 4 * U * ref["top_logprobs"].abs().nan_to_num(0, 0, 0), "top")
    return ref


def inputs(device, rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device=device) * scale
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    return x.to(dtype), t


def plain_gradient(ref, tokens, vocab, temperature, gl, gh, gz, gt, top_ids):
    """The formula in float64, and the bound of the kernel's error before its last rounding."""
    p, logp = ref["p"], torch.where(ref["p"] > 0, ref["logp"], 0.0)
    h = ref["entropy"]
    has = ref["has"] if tokens is not None else torch.zeros_like(ref["bad"])
    g1 = torch.where(has, gl, 0.0) if gl is not None else torch.zeros_like(h)
    even = (gz if gz is not None else 0.0) - g1
    slope = gh if gh is not None else torch.zeros_like(h)
    listed = torch.zeros_like(h)
    if gt is not None:
        gt = torch.where(top_ids >= 0, gt, 0.0)
        even = even - gt.sum(1)
        listed = gt.abs().sum(1)
    bracket = even[:, None] - slope[:, None] * (logp + h[:, None])
    dx = p * bracket
    alone = torch.zeros_like(dx)
    if tokens is not None:
        alone.scatter_add_(1, torch.where(has, tokens, 0).long()[:, None], g1[:, None])
    if gt is not None:
        alone.scatter_add_(1, top_ids.clamp_min(0), gt)
    dx = (dx + alone) / temperature
    es, eh = bounds(ref, vocab)
    d = torch.where(p > 0, ref["d"].abs(), 0.0)
    ep = 2.0 ** -22 + (3 * d + 2 * ref["log_s"].abs()[:, None]) * U + es[:, None]
    size = even.abs() + listed + g1.abs() + (gz.abs() if gz is not None else 0.0) + slope.abs() * h
    eb = (40 * U) * size[:, None] + slope.abs()[:, None] * (eh[:, None] + es[:, None] + 6 * U * (d + logp.abs()))
    tol = p * (ep * bracket.abs() + eb) + (40 * U) * alone.abs() + 40 * U * dx.abs() * temperature
    tol = tol / temperature + 2.0 ** -120
    dead = ref["none"][:, None].expand_as(dx)
    dx = torch.where(dead, 0.0, dx)
    dx = torch.where(ref["bad"][:, None], math.nan, dx)
    return dx, torch.where(dead | ref["bad"][:, None], 0.0, tol)


def check_gradient(grad, dx, tol, dtype):
    got = grad.double()
    assert torch.equal(torch.isnan(got), torch.isnan(dx))
    ok = ~torch.isnan(dx)
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126  # half a subnormal step
    bound = tol * (1 + half) + half * dx.abs() + tiny
    err = (got - dx).abs()[ok] - bound[ok]
    assert float(err.max()) <= 0, float(err.max())


# ------------------------------------------------------------------ CPU: refusals


def _args(**kw):
    base = dict(logits=0x10000, logits_row_stride=64, tokens=0x20000, logits_dtype=N.DTYPE_BF16, tokens_dtype=N.IDS_I64,
                rows=4, vocab=64, top_n=2, temperature=1.0, out_logprobs=0x30000, out_entropy=0x31000, out_lse=0x32000,
                out_top_ids=0x33000, out_top_logprobs=0x34000, out_stats=0x35000, out_status=0x36000)
    return N.sized(N.MtrLogprobArgs, **{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(tokens=None, out_logprobs=None), N.OK), (dict(rows=0, logits=None), N.OK),
    (dict(top_n=0, out_top_ids=None, out_top_logprobs=None), N.OK),
    (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(vocab=0), N.ERR_BAD_SHAPE), (dict(vocab=N.MAX_VOCAB + 1), N.ERR_BAD_SHAPE),
    (dict(logits_row_stride=63), N.ERR_BAD_SHAPE), (dict(logits=None), N.ERR_NULL_ARG), (dict(tokens=None), N.ERR_NULL_ARG),
    (dict(out_top_ids=None), N.ERR_NULL_ARG), (dict(out_top_logprobs=None), N.ERR_NULL_ARG),
    (dict(top_n=33), N.ERR_BAD_PARAM), (dict(top_n=-1), N.ERR_BAD_PARAM), (dict(temperature=0.0), N.ERR_BAD_PARAM),
    (dict(temperature=-1.0), N.ERR_BAD_PARAM), (dict(temperature=math.nan), N.ERR_BAD_PARAM),
    (dict(temperature=math.inf), N.ERR_BAD_PARAM), (dict(temperature=1e-39), N.ERR_BAD_PARAM),
    (dict(logits_dtype=3), N.ERR_BAD_PARAM), (dict(tokens_dtype=2), N.ERR_BAD_PARAM),
    (dict(logits=0x10001), N.ERR_ALIGNMENT), (dict(tokens=0x20004), N.ERR_ALIGNMENT), (dict(out_stats=0x35008), N.ERR_ALIGNMENT),
    (dict(out_logprobs=0x30002), N.ERR_ALIGNMENT), (dict(struct_size=8), N.ERR_ABI), (dict(abi_version=1), N.ERR_ABI),
])
def test_forward_arguments_are_checked_on_the_host(kw, code):
    import ctypes

    a = _args()
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_logprob_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:  # the launcher checks first: no CUDA call
        assert lib.mtr_logprob_launch(ctypes.byref(a), None) == code


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0), N.OK), (dict(stats=None), N.ERR_NULL_ARG), (dict(grad_logits=None), N.ERR_NULL_ARG),
    (dict(tokens=None), N.ERR_NULL_ARG), (dict(top_n=2), N.ERR_NULL_ARG), (dict(grad_row_stride=63), N.ERR_BAD_SHAPE),
    (dict(grad_logits=0x10000), N.ERR_BAD_PARAM), (dict(grad_logits=0x10000 + 4 * 64 * 2 - 2), N.ERR_BAD_PARAM),
    (dict(grad_logits=0x10000 + 4 * 64 * 2), N.OK), (dict(grad_logits=0x50001), N.ERR_ALIGNMENT),
    (dict(stats=0x35004), N.ERR_ALIGNMENT), (dict(temperature=0.0), N.ERR_BAD_PARAM), (dict(struct_size=0), N.ERR_ABI),
])
def test_gradient_arguments_are_checked_on_the_host(kw, code):
    import ctypes

    a = N.sized(N.MtrLogprobGradArgs, logits=0x10000, logits_row_stride=64, tokens=0x20000, logits_dtype=N.DTYPE_BF16,
                tokens_dtype=N.IDS_I64, rows=4, vocab=64, top_n=0, temperature=1.0, stats=0x35000, g_logprobs=0x36000,
                grad_logits=0x50000, grad_row_stride=64)
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_logprob_grad_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_logprob_grad_launch(ctypes.byref(a), None) == code


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 8))
    with pytest.raises(ValueError):
        token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        token_logprobs_backward(x, None, TokenLogprobs(None, None, None, None, None, None))


def test_formula_against_differences():
    # the gradient that the kernel tests use, against central differences of the definition (CPU, float64)
    rows, vocab, temp = 4, 23, 0.7
    g = torch.Generator().manual_seed(3)
    x = torch.randn((rows, vocab), generator=g, dtype=torch.float64) * 2
    x[1, 5:20] = -math.inf
    tokens = torch.tensor([3, 2, -100, 22])
    gl, gh, gz = (torch.randn(rows, generator=g, dtype=torch.float64) for _ in range(3))
    gt = torch.randn((rows, 3), generator=g, dtype=torch.float64)
    ref = reference(x, tokens, 3, temp)
    dx, _ = plain_gradient(ref, tokens, vocab, temp, gl, gh, gz, gt, ref["top_ids"])

    def value(y):
        r = reference(y, tokens, 3, temp)
        top = r["logp"].gather(1, ref["top_ids"])
        return (gl * r["logprobs"] + gh * r["entropy"] + gz * r["lse"] + (gt * top).sum(1)).sum()

    for r in range(rows):
        for v in range(vocab):
            if x[r, v] == -math.inf:
                assert dx[r, v] == 0
                continue
            e = torch.zeros_like(x)
            e[r, v] = 1e-5
            assert abs(float((value(x + e) - value(x - e)) / 2e-5) - float(dx[r, v])) < 1e-7  # h^2 f''' / 6 plus 1e-15 / h


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top_n", [
    (1, 1, 0), (1, 1, 3), (3, 2, 2), (5, 7, 8), (2, 31, 5), (4, 33, 1), (3, 255, 20), (7, 257, 32), (130, 1000, 5), (64, 4096, 8),
    (9, 4099, 20), (500, 4096, 0), (5, 8192, 32), (3, 32771, 8), (20, 65536, 1), (2, 131072, 32), (1, 131071, 5), (300, 5000, 4),
    (2500, 300, 32), (2400, 4096, 30), (2400, 2100, 4), (1300, 9000, 28), (40, 131072, 25)])
def test_forward(cuda_device, dtype, rows, vocab, top_n):
    logits, tokens = inputs(cuda_device, rows, vocab, dtype, seed=rows + vocab)
    check_forward(token_logprobs(logits, tokens, top_n=top_n), logits, tokens, top_n)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 3.0])
def test_temperature_and_int32_tokens(cuda_device, dtype, temperature):
    logits, tokens = inputs(cuda_device, 12, 700, dtype, seed=4)
    r = token_logprobs(logits, tokens.int(), top_n=6, temperature=temperature)
    # 1 / T is rounded: |x| 2^-24 more in the log-sum-exp, which 2 2^-24 |lse| covers
    check_forward(r, logits, tokens, 6, temperature)


def _odd_rows(device, dtype, vocab):
    """Rows that a mask empties in part or whole, ties, signed zeros, extremes, and values that are not numbers."""
    low = torch.finfo(dtype).min
    x, t = inputs(device, 17, vocab, dtype, seed=9)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, vocab - 1] = 2.5
    x[2] = low
    x[3, : vocab // 2] = low
    x[4] = 1.25
    x[5, ::2] = 0.0
    x[5, 1::2] = -0.0
    x[6, vocab // 3] = math.nan
    x[7, vocab // 2] = math.inf
    x[8] = -math.inf
    x[8, 0] = math.nan
    x[9] = torch.arange(vocab, device=device).to(dtype) * 2.0 ** -8
    x[10] = -torch.arange(vocab, device=device).to(dtype) * 2.0 ** -8
    x[11] = torch.finfo(dtype).max
    x[12] = -math.inf
    x[12, : min(3, vocab)] = low
    x[13] = 0.0
    x[13, vocab // 2] = 60.0
    x[14] = -math.inf
    x[14, vocab // 2:] = 1.0
    x[15, 0] = math.inf
    x[15, vocab - 1] = math.nan
    t[13] = vocab // 2
    return x, t


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top_n", [(2, 2), (40, 3), (1000, 32), (4096, 20), (9001, 7), (70000, 32)])
def test_rows_that_masks_and_values_make_odd(cuda_device, dtype, vocab, top_n):
    x, t = _odd_rows(cuda_device, dtype, vocab)
    status = torch.zeros(17, dtype=torch.int32, device=cuda_device)
    t[16] = vocab + 3
    r = token_logprobs(x, t, top_n=top_n, status=status)
    ref = check_forward(r, x, t, top_n)
    want = torch.where(ref["bad"], N.ROW_NONFINITE, torch.where(ref["none"], N.ROW_ALL_MASKED, 0))
    want[16] |= N.ROW_BAD_ID
    assert torch.equal(status.long(), want)
    assert S.row_status_report(status)["bad_id"] == [16]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top_n", [(3, 131072, 32), (2, 65536, 3), (2400, 4096, 32), (150, 20000, 20)])
def test_alternatives_where_candidates_crowd(cuda_device, dtype, rows, vocab, top_n):
    # few distinct values, many ties at the bound, and rows whose largest logits all lie in one thread's vectors
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    x = torch.randint(0, 4, (rows, vocab), generator=g, device=cuda_device).float()
    x[1] = 0.5
    x[0] = torch.arange(vocab, device=cuda_device) * 2.0 ** -7
    for step in (32 * 8, 32 * 4, 128 * 8, 128 * 4, 256 * 8, 256 * 4):  # the stride of a thread's vectors, by warps and type
        if step < vocab:
            x[rows - 1, ::step] = 5.0
            x[rows - 1, 1::step] = 6.0
    x = x.to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda_device)
    check_forward(token_logprobs(x, t, top_n=top_n), x, t, top_n)


@gpu
def test_small_entropies_keep_their_digits(cuda_device):
    # nearly all mass on one id: log p and the entropy are small numbers, known from log1p
    x = torch.zeros((3, 64), device=cuda_device)
    x[0, 5], x[1, 6], x[2, 7] = 12.0, 16.0, 20.0
    t = torch.tensor([5, 6, 7], device=cuda_device)
    r = token_logprobs(x, t)
    ref = reference(x, t, 0)
    assert float(((r.logprobs.double() - ref["logprobs"]) / ref["logprobs"]).abs().max()) < 2.0 ** -20
    assert float(((r.entropy.double() - ref["entropy"]) / ref["entropy"]).abs().max()) < 2.0 ** -20


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride,offset", [(100, 101, 1), (4096, 4099, 3), (4095, 4095, 5), (20000, 20003, 7), (8193, 8193, 1),
                                                 (2049, 2049, 0), (4097, 4097, 2)])
def test_strided_rows_off_any_boundary(cuda_device, dtype, vocab, stride, offset):
    rows = 11
    x, t = inputs(cuda_device, rows, vocab, dtype, seed=5)
    t[::2] = vocab - 1
    t[1] = 0
    wide = torch.full((rows * stride + offset,), math.nan, dtype=dtype, device=cuda_device)  # what is not the row's is not read
    view = wide[offset:].as_strided((rows, vocab), (stride, 1))
    view.copy_(x)
    a, b = token_logprobs(view, t, top_n=9), token_logprobs(x, t, top_n=9)
    check_forward(a, x, t, 9)
    assert torch.equal(a.top_ids, b.top_ids)
    g = torch.rand(rows, device=cuda_device)
    out = torch.full((rows, stride), 7.0, dtype=dtype, device=cuda_device)
    token_logprobs_backward(view, t, a, grad_logprobs=g, out=out[:, :vocab])
    ref = reference(x, t, 0)
    dx, tol = plain_gradient(ref, t, vocab, 1.0, g.double(), None, None, None, None)
    check_gradient(out[:, :vocab], dx, tol, dtype)
    assert bool((out[:, vocab:] == 7.0).all())  # columns behind the vocabulary stay


@gpu
def test_no_tokens_no_rows_and_padding(cuda_device):
    x, t = inputs(cuda_device, 6, 300, torch.bfloat16)
    check_forward(token_logprobs(x, None, top_n=4), x, None, 4)
    t[1], t[3] = -1, -100
    r = token_logprobs(x, t)
    check_forward(r, x, t, 0)
    assert r.logprobs[1] == 0 and r.logprobs[3] == 0
    e = token_logprobs(x[:0], t[:0], top_n=3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)
    assert token_logprobs_backward(x[:0], t[:0], e, grad_logprobs=e.logprobs).shape == (0, 300)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top_n,temperature", [
    (1, 1, 1, 1.0), (3, 2, 0, 1.0), (5, 37, 5, 0.7), (64, 4096, 8, 1.0), (7, 4099, 32, 1.5), (3, 70001, 3, 1.0), (2, 131072, 0, 0.9),
    (400, 513, 2, 1.0)])
def test_gradient(cuda_device, dtype, rows, vocab, top_n, temperature):
    x, t = inputs(cuda_device, rows, vocab, dtype, seed=vocab)
    if rows > 2:
        x[1, vocab // 2:] = -math.inf
        t[1], t[2] = 0, -100
    g = torch.Generator(device=cuda_device).manual_seed(1)
    gl, gh, gz = (torch.randn(rows, generator=g, device=cuda_device) for _ in range(3))
    gt = torch.randn((rows, top_n), generator=g, device=cuda_device)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top_n=top_n, temperature=temperature)
    outs, gs = [r.logprobs, r.entropy, r.lse], [gl, gh, gz]
    if top_n:
        # a missing alternative's log probability is -inf: nothing flows from it
        outs.append(r.top_logprobs)
        gs.append(gt)
    torch.autograd.backward(outs, gs)
    ref = reference(x, t, top_n, temperature)
    dx, tol = plain_gradient(ref, t, vocab, temperature, gl.double(), gh.double(), gz.double(), gt.double() if top_n else None,
                             ref["top_ids"])
    check_gradient(leaf.grad, dx, tol, dtype)
    assert not r.top_ids.requires_grad and not r.stats.requires_grad


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 4096, 9001])
def test_gradient_of_odd_rows(cuda_device, dtype, vocab):
    x, t = _odd_rows(cuda_device, dtype, vocab)
    t[16] = vocab  # outside: no token
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top_n=4)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    gl, gh, gz = (torch.randn(17, generator=g, device=cuda_device) for _ in range(3))
    gt = torch.randn((17, 4), generator=g, device=cuda_device)
    (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.lse, r.top_logprobs), leaf, (gl, gh, gz, gt))
    ref = reference(x, t, 4)
    dx, tol = plain_gradient(ref, t, vocab, 1.0, gl.double(), gh.double(), gz.double(), gt.double(), ref["top_ids"])
    check_gradient(grad, dx, tol, dtype)


@gpu
def test_gradient_parts_alone_and_expanded(cuda_device):
    x, t = inputs(cuda_device, 30, 513, torch.float32, seed=8)
    ref = reference(x, t, 5)
    ones = torch.ones(30, dtype=torch.float64, device=cuda_device)
    for part in ("logprobs", "entropy", "lse", "top_logprobs"):
        leaf = x.clone().requires_grad_(True)
        getattr(token_logprobs(leaf, t, top_n=5), part).sum().backward()  # an expanded scalar
        gt = torch.ones((30, 5), dtype=torch.float64, device=cuda_device) if part == "top_logprobs" else None
        dx, tol = plain_gradient(ref, t, 513, 1.0, ones if part == "logprobs" else None, ones if part == "entropy" else None,
                                 ones if part == "lse" else None, gt, ref["top_ids"])
        check_gradient(leaf.grad, dx, tol, torch.float32)
    leaf = x.clone().requires_grad_(True)  # without tokens
    r = token_logprobs(leaf)
    assert r.logprobs is None
    r.entropy.sum().backward()
    dx, tol = plain_gradient(reference(x, None, 0), None, 513, 1.0, None, ones, None, None, None)
    check_gradient(leaf.grad, dx, tol, torch.float32)
    with torch.no_grad():
        assert not token_logprobs(leaf, t).logprobs.requires_grad


@gpu
def test_refusals(cuda_device):
    x, t = inputs(cuda_device, 4, 64, torch.float32)
    for bad, exc in ((lambda: token_logprobs(x.double(), t), TypeError), (lambda: token_logprobs(x[0], t), ValueError),
                     (lambda: token_logprobs(x.T, t), ValueError), (lambda: token_logprobs(x, t[:3]), ValueError),
                     (lambda: token_logprobs(x, t.float()), TypeError), (lambda: token_logprobs(x, t.cpu()), ValueError),
                     (lambda: token_logprobs(x, t, top_n=33), ValueError), (lambda: token_logprobs(x, t, top_n=-1), ValueError),
                     (lambda: token_logprobs(x, t, temperature=0.0), ValueError),
                     (lambda: token_logprobs(x[:, :0], t), ValueError),
                     (lambda: token_logprobs(x[:1].expand(4, 64), t), ValueError),
                     (lambda: token_logprobs(x, t, status=torch.zeros(4, device=cuda_device)), ValueError),
                     (lambda: token_logprobs_backward(x, t, token_logprobs(x, t), grad_logprobs=t.float(), out=x), ValueError),
                     (lambda: token_logprobs_backward(x, t, token_logprobs(x, t), grad_logprobs=t.double()), ValueError),
                     (lambda: token_logprobs_backward(x, t, token_logprobs(x[:3], t[:3]), grad_lse=t.float()), ValueError),
                     (lambda: token_logprobs_backward(x, None, token_logprobs(x), grad_logprobs=t.float()), ValueError)):
        with pytest.raises(exc):
            bad()


@gpu
def test_same_bits_again_on_another_stream_and_in_graphs(cuda_device):
    x, t = inputs(cuda_device, 200, 5000, torch.bfloat16, seed=6)
    g = torch.rand(200, device=cuda_device)

    def both():
        r = token_logprobs(x, t, top_n=7)
        return list(r) + [token_logprobs_backward(x, t, r, grad_logprobs=g, grad_entropy=g, grad_top_logprobs=r.top_logprobs)]

    want = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    x2, _ = inputs(cuda_device, 200, 5000, torch.bfloat16, seed=7)
    x.copy_(x2)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    new = both()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(new, out))
    assert not torch.equal(new[0], want[0])


@gpu
@pytest.mark.parametrize("do_sample", [True, False])
def test_sampler_scores_its_tokens(cuda_device, do_sample):
    rows, vocab = 48, 4096
    x, _ = inputs(cuda_device, rows, vocab, torch.bfloat16, seed=11)
    kw = dict(vocab_size=vocab, num_rows=rows, device=cuda_device, temperature=0.9, top_k=50, do_sample=do_sample,
              eos_token_ids=range(8), eos_ranges=[(0, 2048)], pad_token_id=1, track_finished=True, return_scores=True)
    a, b = S.FusedSampler(**kw), S.FusedSampler(**kw, token_logprobs=3)
    for step in range(3):
        u = torch.rand(rows, device=cuda_device)
        done = a.unfinished == 0
        ids = a.step(x, uniforms=u)
        assert torch.equal(ids, b.step(x, uniforms=u)) and torch.equal(a.scores, b.scores)
        given = torch.where(done, -1, ids)
        check_forward(b.token_logprobs, a.scores, given, 3)
        assert bool((b.token_logprobs.logprobs[done] == 0).all())
    assert bool(done.any()) and a.token_logprobs is None
    with pytest.raises(ValueError):
        S.FusedSampler(**kw, token_logprobs=40)


# ------------------------------------------------------------------ gradients that are small beside their terms


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.5])
@pytest.mark.parametrize("top_n", [0, 3])
def test_small_gradients_keep_their_digits(cuda_device, dtype, temperature, top_n):
    # A given token that has nearly all the mass: its gradient g (1 - p) / T is far smaller than g / T.  With 63 zeros beside
    # logit / T = 12, 16, 20 every term is positive.  Relative errors: a term of S' 2^-22 + 3 2^-24 |d|, |d| <= 20; its sum, log1p
    # and expm1 below 70 2^-24 more; d and its mean, products: 10 2^-24.  In all less than (4 + 60 + 70 + 10) 2^-24 < 2^-16.
    x = torch.zeros((3, 64), device=cuda_device)
    x[0, 5], x[1, 6], x[2, 7] = 12.0 * temperature, 16.0 * temperature, 20.0 * temperature
    x = x.to(dtype)
    t = torch.tensor([5, 6, 7], device=cuda_device)
    r = token_logprobs(x, t, top_n=top_n, temperature=temperature)
    gl = torch.full((3,), 1.5, device=cuda_device)
    gh, gz = torch.full((3,), -0.25, device=cuda_device), torch.zeros(3, device=cuda_device)
    gt = torch.zeros((3, top_n), device=cuda_device)
    gt[:, :1] = 0.5  # the first alternative is the token
    grad = token_logprobs_backward(x, t, r, grad_logprobs=gl, grad_entropy=gh, grad_lse=gz, temperature=temperature,
                                   grad_top_logprobs=gt if top_n else None)
    xd = x.double() / temperature
    far = xd.amax(1)  # of each other id from the token
    rest = 63 * torch.exp(-far)  # S - 1
    logp = -torch.log1p(rest)
    one_less_p = -torch.expm1(logp)
    p = torch.exp(logp)
    entropy = -p * logp + rest * p * (far - logp)
    own = 1.5 + (0.5 if top_n else 0.0)
    want = (own * one_less_p + 0.25 * p * (logp + entropy)) / temperature
    got = grad[torch.arange(3, device=cuda_device), t].double()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0  # the fp32 rounding is in the count above
    err = ((got - want) / want).abs()
    assert float(err.max()) <= 2.0 ** -16 * (1 + half) + half, err


# ------------------------------------------------------------------ forward-mode derivatives


def _refuses_tangents(device):
    import torch.autograd.forward_ad as fwd

    x, t = torch.randn((3, 20), device=device), torch.tensor([1, 2, 3], device=device)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(dual, t)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(dual, t)
        result = TokenLogprobs(None, x[:, 0], x[:, 0], t[:, None][:, :0], x[:, :0], x[:, :4].contiguous())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs_backward(dual, t, result, grad_lse=x[:, 0].contiguous())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs_backward(x, t, result, grad_lse=fwd.make_dual(x[:, 0].contiguous(), torch.ones(3, device=device)))


def test_forward_mode_is_refused():
    _refuses_tangents("cpu")


@gpu
def test_forward_mode_is_refused_and_plain_tensors_pass(cuda_device):
    import torch.autograd.forward_ad as fwd

    _refuses_tangents(cuda_device)
    x, t = inputs(cuda_device, 5, 70, torch.float32)
    want = token_logprobs(x, t)
    with fwd.dual_level():
        assert torch.equal(token_logprobs(x, t).logprobs, want.logprobs)


# ------------------------------------------------------------------ logits and gradient side by side in one buffer


@pytest.mark.parametrize("at,code", [(64, N.OK), (63, N.ERR_BAD_PARAM), (150 - 64, N.OK), (150 - 63, N.ERR_BAD_PARAM), (-64, N.OK)])
def test_logits_and_gradient_may_share_a_buffer_of_wider_rows(at, code):
    import ctypes

    a = N.sized(N.MtrLogprobGradArgs, logits=0x10000, logits_row_stride=150, tokens=0x20000, logits_dtype=N.DTYPE_BF16,
                tokens_dtype=N.IDS_I64, rows=4, vocab=64, top_n=0, temperature=1.0, stats=0x35000, g_logprobs=0x36000,
                grad_logits=0x10000 + 2 * at, grad_row_stride=150)
    assert N.load().mtr_logprob_grad_validate(ctypes.byref(a)) == code


@gpu
@pytest.mark.parametrize("gap", [0, 3])
def test_logits_and_gradient_in_one_buffer(cuda_device, gap):
    rows, vocab = 40, 1000
    x, t = inputs(cuda_device, rows, vocab, torch.bfloat16, seed=22)
    both = torch.full((rows, 2 * vocab + gap), 7.0, dtype=torch.bfloat16, device=cuda_device)
    both[:, :vocab] = x
    g = torch.rand(rows, device=cuda_device)
    logits, grad = both[:, :vocab], both[:, vocab + gap:]
    token_logprobs_backward(logits, t, token_logprobs(logits, t), grad_logprobs=g, grad_lse=g, out=grad)
    assert torch.equal(grad, token_logprobs_backward(x, t, token_logprobs(x, t), grad_logprobs=g, grad_lse=g))
    assert torch.equal(logits, x) and bool((both[:, vocab:vocab + gap] == 7.0).all())


# ------------------------------------------------------------------ logits further apart than the type's largest value


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 2.0 ** 100])
@pytest.mark.parametrize("vocab", [5, 700, 70000])
def test_logits_at_both_ends_of_the_range(cuda_device, dtype, temperature, vocab):
    # x - max passes the range before the division by T brings it back
    x = torch.zeros((4, vocab), device=cuda_device)
    x[0, 0], x[0, 1], x[0, 2] = 3.0e38, -3.0e38, 2.0e38
    x[1] = -3.0e38
    x[1, vocab - 1] = 3.0e38
    x[2, ::2] = 1.0e38
    x[2, 1::2] = -2.5e38
    x[3, 3] = -math.inf
    x[3, 4] = torch.finfo(dtype).max
    x = x.to(dtype)
    t = torch.tensor([1, 0, 1, 4], device=cuda_device)
    r = token_logprobs(x, t, top_n=4, temperature=temperature)
    ref = reference(x, t, 4, temperature)
    f32 = lambda v: v.float().double()  # noqa: E731  a log probability below the fp32 range reads -inf
    es, eh = bounds(ref, vocab)
    close(r.logprobs, f32(ref["logprobs"]), es + 4 * U * ref["logprobs"].abs(), "logprobs")
    close(r.entropy, ref["entropy"], eh, "entropy")
    close(r.lse, ref["lse"], es + 2 * U * ref["lse"].abs(), "lse")
    assert torch.equal(r.top_ids, ref["top_ids"])
    close(r.top_logprobs, f32(ref["top_logprobs"]), es[:, None] + 4 * U * ref["top_logprobs"].abs().nan_to_num(0, 0, 0), "top")
    g = torch.tensor([1.0, -2.0, 0.5, 3.0], device=cuda_device) * temperature
    grad = token_logprobs_backward(x, t, r, grad_logprobs=g, grad_entropy=g, grad_lse=-g, temperature=temperature)
    dx, tol = plain_gradient(ref, t, vocab, temperature, g.double(), g.double(), -g.double(), None, None)
    check_gradient(grad, dx, tol, dtype)


@pytest.mark.parametrize("temperature,code", [(2.0 ** 100, N.OK), (2.0 ** 100 * (1 + 2.0 ** -23), N.ERR_BAD_PARAM), (3.0e38, N.ERR_BAD_PARAM)])
def test_largest_temperature(temperature, code):
    import ctypes

    a = _args(temperature=temperature)
    assert N.load().mtr_logprob_validate(ctypes.byref(a)) == code
    if code != N.OK:
        assert N.load().mtr_logprob_launch(ctypes.byref(a), None) == code
