"""The 8-bit output projection.  Everything before the last rounding is defined
to the bit (the quantisation, the exact integer sum, three fp32 roundings), so
the logits are compared for equality with the definition evaluated in float64
and float32 by elementary operations."""

import ctypes
import math

import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.int8_head import Int8Weight, lm_head_logits_int8, quantize_rows
from mapperatorinator_b200.scoring import token_logprobs

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain_quantize(x):
    x = x.float().cpu()
    top = x.abs().amax(1)
    bad = ~torch.isfinite(x).all(1)
    scale = torch.where(bad, math.nan, top * torch.tensor(1 / 127, dtype=torch.float32))
    q = torch.where((scale > 0)[:, None], x / scale[:, None], 0.0)
    return torch.round(q.nan_to_num(0.0)).to(torch.int8), scale


def plain_logits(q, scale, wq, ws, dtype):
    acc = (q.double() @ wq.double().T).float()  # exact sums below 2^53, then one rounding
    return ((acc * scale[:, None]) * ws[None, :]).to(dtype)


def inputs(device, rows, d, vocab, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    h = torch.randn((rows, d), generator=g, device=device).to(dtype)
    w = torch.randn((vocab, d), generator=g, device=device) * 0.02
    return h, w


def same(got, want):
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan]), int((got[~nan] != want[~nan]).sum())


# ------------------------------------------------------------------ CPU


def _quant_args(**kw):
    base = dict(x=0x100000, x_row_stride=64, x_dtype=N.DTYPE_BF16, rows=4, cols=64, q=0x200000, q_row_stride=64, scale=0x300000)
    return N.sized(N.MtrQuantizeArgs, **{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0, x=None), N.OK), (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(cols=0), N.ERR_BAD_SHAPE),
    (dict(cols=N.MAX_I8_D_MODEL + 1), N.ERR_BAD_SHAPE),
    (dict(x_row_stride=63), N.ERR_BAD_SHAPE), (dict(q_row_stride=63), N.ERR_BAD_SHAPE), (dict(x_dtype=5), N.ERR_BAD_PARAM),
    (dict(q=None), N.ERR_NULL_ARG), (dict(scale=None), N.ERR_NULL_ARG), (dict(x=0x100001), N.ERR_ALIGNMENT),
    (dict(scale=0x300002), N.ERR_ALIGNMENT), (dict(q=0x100010), N.ERR_BAD_PARAM), (dict(struct_size=1), N.ERR_ABI)])
def test_quantize_arguments_are_checked_on_the_host(kw, code):
    a = _quant_args()
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_quantize_rows_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_quantize_rows_launch(ctypes.byref(a), None) == code


def _proj_args():
    return N.sized(N.MtrLmHeadI8Args, hidden=0x1000000, hidden_row_stride=100, weight=0x2000000, weight_row_stride=112,
                   weight_scale=0x3000000, logits=0x4000000, logits_row_stride=77, hidden_dtype=N.DTYPE_BF16,
                   logits_dtype=N.DTYPE_BF16, rows=900, d_model=100, vocab=77, workspace=0x5000000, workspace_bytes=1 << 20)


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0, hidden=None), N.OK), (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(rows=N.MAX_I8_ROWS + 1), N.ERR_BAD_SHAPE),
    (dict(d_model=0), N.ERR_BAD_SHAPE), (dict(d_model=N.MAX_I8_D_MODEL + 1), N.ERR_BAD_SHAPE), (dict(vocab=0), N.ERR_BAD_SHAPE),
    (dict(vocab=N.MAX_VOCAB + 1), N.ERR_BAD_SHAPE), (dict(hidden_dtype=3), N.ERR_BAD_PARAM), (dict(logits_dtype=-1), N.ERR_BAD_PARAM),
    (dict(weight=None), N.ERR_NULL_ARG), (dict(weight_scale=None), N.ERR_NULL_ARG), (dict(workspace=None), N.ERR_NULL_ARG),
    (dict(workspace_bytes=900 * 112), N.ERR_BAD_SHAPE), (dict(rows=8, workspace=None, workspace_bytes=0), N.OK),
    (dict(workspace=0x5000010), N.ERR_ALIGNMENT),
    (dict(weight_row_stride=104), N.ERR_ALIGNMENT), (dict(weight=0x2000008), N.ERR_ALIGNMENT),
    (dict(weight_row_stride=96), N.ERR_BAD_SHAPE), (dict(logits_row_stride=76), N.ERR_BAD_SHAPE),
    (dict(hidden_row_stride=99), N.ERR_BAD_SHAPE), (dict(logits=0x1000000), N.ERR_BAD_PARAM),
    (dict(workspace=0x4000000), N.ERR_BAD_PARAM), (dict(error_word=2), N.ERR_ALIGNMENT), (dict(abi_version=9), N.ERR_ABI)])
def test_projection_arguments_are_checked_on_the_host(kw, code):
    a = _proj_args()
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_lmhead_i8_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_lmhead_i8_launch(ctypes.byref(a), None) == code


def test_projection_and_sampler_must_share_the_logits():
    lm, a = _proj_args(), N.new_args()
    a.logits, a.logits_row_stride, a.logits_dtype, a.vocab, a.num_rows = lm.logits, 77, N.DTYPE_BF16, 77, 900
    a.select_mode, a.out_ids = N.SELECT_ARGMAX, 0x6000000
    lib = N.load()
    for field, value, code in (("logits", 0x7000000, N.ERR_BAD_PARAM), ("logits_row_stride", 78, N.ERR_BAD_PARAM),
                               ("logits_dtype", N.DTYPE_F16, N.ERR_BAD_PARAM), ("num_rows", 901, N.ERR_BAD_SHAPE)):
        b = N.MtrSamplerArgs()
        ctypes.pointer(b)[0] = a
        setattr(b, field, value)
        assert lib.mtr_lmhead_i8_sample_launch(ctypes.byref(lm), ctypes.byref(b), None) == code, field
    lm.rows = a.num_rows = 0
    assert lib.mtr_lmhead_i8_sample_launch(ctypes.byref(lm), ctypes.byref(a), None) == N.OK


def test_workspace_sizes():
    assert N.lmhead_i8_workspace(0, 64, 100) == 0 and N.lmhead_i8_workspace(4, 0, 100) == 0
    assert N.lmhead_i8_workspace(3, 100, 4096) == 0  # few rows
    assert N.lmhead_i8_workspace(3, 900, 131072) == 2816 + 12  # 3 rows of 912 bytes, the scales on the next 256-byte boundary
    assert N.lmhead_i8_workspace(301, 100, 77) == 33792 + 1204
    assert N.lmhead_i8_workspace(N.MAX_I8_ROWS, N.MAX_I8_D_MODEL, 1) == (1 << 39) + (1 << 24)


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 16))
    with pytest.raises(ValueError):
        quantize_rows(x)
    with pytest.raises(ValueError):
        lm_head_logits_int8(x, x.to(torch.int8), torch.ones(2))


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (130, 100), (64, 768), (17, 1001), (2, 4096), (3, 70001)])
def test_quantize_rows(cuda_device, dtype, rows, cols):
    x, _ = inputs(cuda_device, rows, cols, 1, dtype, seed=rows + cols)
    q, scale = quantize_rows(x)
    want_q, want_s = plain_quantize(x)
    same(scale, want_s)
    same(q, want_q)
    assert q.stride(0) % 16 == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [40, 1000])
def test_quantize_odd_rows(cuda_device, dtype, cols):
    x, _ = inputs(cuda_device, 10, cols, 1, dtype, seed=3)
    x[0] = 0.0
    x[1, 7] = math.nan
    x[2, 8] = math.inf
    x[3, 9] = -math.inf
    x[4] = torch.finfo(dtype).max
    x[5] = x[5] * torch.finfo(dtype).tiny  # subnormal scales, or none
    x[6] = torch.finfo(dtype).tiny * 0.25 if dtype == torch.float32 else torch.finfo(dtype).smallest_normal
    # halves: every quotient n + 1/2 rounds to even (127 / 127 = 1 is the scale)
    x[7] = (torch.arange(cols, device=cuda_device) % 100 - 50 + 0.5).to(dtype)
    x[7, 0] = 127.0
    x[8] = 0.0
    x[8, cols - 1] = -3.0
    q, scale = quantize_rows(x)
    want_q, want_s = plain_quantize(x)
    same(scale, want_s)
    same(q, want_q)


@gpu
def test_quantize_strided_rows(cuda_device):
    x, _ = inputs(cuda_device, 9, 203, 1, torch.float16, seed=5)
    wide = torch.full((9, 211), math.nan, dtype=torch.float16, device=cuda_device)
    wide[:, 3:206] = x
    q, scale = quantize_rows(wide[:, 3:206])
    want_q, want_s = plain_quantize(x)
    same(q, want_q)
    same(scale, want_s)
    assert quantize_rows(x[:0])[0].shape == (0, 203)


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("rows,d,vocab,dtype", [
    (1, 1, 1, torch.float32), (1, 16, 8, torch.bfloat16), (8, 2048, 1000, torch.bfloat16), (5, 1001, 300, torch.float16),
    (8, 100, 131072, torch.float32), (1, 8192, 77, torch.bfloat16), (1, 8193, 77, torch.bfloat16), (9, 64, 20000, torch.float32),
    (3, 15, 3, torch.bfloat16), (4, 2048, 16000, torch.float32), (8, 513, 131072, torch.bfloat16), (2, 4096, 131072, torch.bfloat16),
    (6, 1000, 999, torch.float16), (1, 65536, 40, torch.bfloat16), (1, 65537, 40, torch.float32), (2, 768, 4096, torch.bfloat16), (128, 768, 4096, torch.bfloat16),
    (33, 100, 77, torch.float16), (129, 1001, 4099, torch.float16), (300, 64, 520, torch.float32), (256, 128, 8192, torch.bfloat16),
    (513, 2048, 1000, torch.bfloat16), (1030, 96, 264, torch.float32), (64, 3000, 131072, torch.bfloat16),
    (300, 2100, 8200, torch.bfloat16), (300, 64, 40000, torch.bfloat16)])
def test_logits_equal_the_definition(cuda_device, out_dtype, rows, d, vocab, dtype):
    h, w = inputs(cuda_device, rows, d, vocab, dtype, seed=rows + d + vocab)
    weight = Int8Weight.from_weight(w)
    out = lm_head_logits_int8(h, weight.q, weight.scale, out_dtype=out_dtype)
    q, scale = plain_quantize(h)
    wq, ws = plain_quantize(w)
    same(weight.q, wq)
    same(out, plain_logits(q.to(cuda_device), scale.to(cuda_device), weight.q, weight.scale, out_dtype))
    assert torch.equal(out, lm_head_logits_int8(h, weight.q, weight.scale, out_dtype=out_dtype))


@gpu
def test_largest_sums_are_exact(cuda_device):
    # |sum| = 127 * 128 * 131072 = 2130706432, near the ends of int32
    d = N.MAX_I8_D_MODEL
    h = torch.ones((3, d), device=cuda_device)
    h[1] = -1.0
    h[2, ::2] = -1.0
    wq = torch.full((9, d), -128, dtype=torch.int8, device=cuda_device)
    wq[4:] = 127
    ws = torch.full((9,), 2.0 ** -10, device=cuda_device)
    out = lm_head_logits_int8(h, wq, ws, out_dtype=torch.float32)
    q, scale = quantize_rows(h)
    same(out, plain_logits(q, scale, wq, ws, torch.float32))


@gpu
@pytest.mark.parametrize("rows", [7, 147])
def test_odd_rows_and_weights(cuda_device, rows):
    h, w = inputs(cuda_device, 7, 200, 300, torch.bfloat16, seed=2)
    h[1], h[2, 5], h[3, 6] = 0.0, math.nan, math.inf
    w[4] = 0.0
    h = torch.cat([h] * (rows // 7))
    weight = Int8Weight.from_weight(w)
    out = lm_head_logits_int8(h, weight.q, weight.scale)
    q, scale = quantize_rows(h)
    same(out, plain_logits(q, scale, weight.q, weight.scale, torch.bfloat16))
    assert bool(torch.isnan(out[2:4]).all()) and bool((out[1] == 0).all()) and bool((out[0, 4:5] == 0).all())


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride,offset", [(300, 301, 1), (256, 260, 0), (4096, 4104, 8), (4099, 4100, 2), (4099, 4104, 0),
                                                 (29, 32, 8), (4102, 4104, 0), (3, 8, 0)])
def test_strides_and_what_lies_behind(cuda_device, out_dtype, vocab, stride, offset):
    rows, d = 140, 200
    h, w = inputs(cuda_device, rows, d, vocab, seed=6)
    wide_h = torch.full((rows, 300), math.nan, dtype=torch.bfloat16, device=cuda_device)
    wide_h[:, 51:251] = h
    weight = Int8Weight.from_weight(w)
    wide_w = torch.full((vocab, 256), 99, dtype=torch.int8, device=cuda_device)
    wide_w[:, :d] = weight.q
    buf = torch.full((offset + (rows + 3) * stride,), 7.0, dtype=out_dtype, device=cuda_device)
    out = buf[offset:].as_strided((rows, vocab), (stride, 1))
    got = lm_head_logits_int8(wide_h[:, 51:251], wide_w[:, :d], weight.scale, out)
    assert got is out
    assert torch.equal(out, lm_head_logits_int8(h, weight.q, weight.scale, out_dtype=out_dtype))
    few_buf = torch.full((offset + 9 * stride,), 7.0, dtype=out_dtype, device=cuda_device)
    few = few_buf[offset:].as_strided((7, vocab), (stride, 1))
    lm_head_logits_int8(wide_h[:7, 51:251], wide_w[:, :d], weight.scale, few)  # few rows: another kernel, the same bits
    assert torch.equal(out[:7], few)
    rest = torch.ones_like(few_buf, dtype=torch.bool)
    rest[offset:].as_strided((7, vocab), (stride, 1)).fill_(False)
    assert bool((few_buf[rest] == 7.0).all())
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[offset:].as_strided((rows, vocab), (stride, 1)).fill_(False)
    assert bool((buf[rest] == 7.0).all())  # columns behind the vocabulary and rows behind the last


@gpu
def test_refusals(cuda_device):
    h, w = inputs(cuda_device, 4, 64, 80)
    q, s = quantize_rows(w)
    odd = torch.zeros((80, 65), dtype=torch.int8, device=cuda_device)[:, :64]
    for bad, exc in ((lambda: lm_head_logits_int8(h[:, :32], q, s), ValueError), (lambda: lm_head_logits_int8(h.double(), q, s), TypeError),
                     (lambda: lm_head_logits_int8(h, q.float(), s), TypeError), (lambda: lm_head_logits_int8(h, q, s[:79]), ValueError),
                     (lambda: lm_head_logits_int8(h, q, s.double()), ValueError), (lambda: lm_head_logits_int8(h, odd, s), ValueError),
                     (lambda: lm_head_logits_int8(h, q, s.cpu()), ValueError), (lambda: lm_head_logits_int8(h.T, q, s), ValueError),
                     (lambda: lm_head_logits_int8(h, q, s, h), ValueError),
                     (lambda: lm_head_logits_int8(h, q, s, out_dtype=torch.int32), TypeError),
                     (lambda: quantize_rows(h[:, :0]), ValueError), (lambda: quantize_rows(h.long()), TypeError)):
        with pytest.raises(exc):
            bad()
    assert lm_head_logits_int8(h[:0], q, s).shape == (0, 80)


@gpu
@pytest.mark.parametrize("rows", [2, 130])
def test_streams_and_graphs(cuda_device, rows):
    h, w = inputs(cuda_device, 130, 768, 1000, seed=9)
    weight = Int8Weight.from_weight(w)
    call = lambda: lm_head_logits_int8(h[:rows], weight.q, weight.scale)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(3)]
    here = [call() for _ in range(3)]  # two streams at once, a workspace each
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in other + here)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    h.copy_(inputs(cuda_device, 130, 768, 1000, seed=10)[0])
    for graph, _ in graphs:
        graph.replay()
    new = call()
    torch.cuda.synchronize()
    assert all(torch.equal(new, o) for _, o in graphs) and not torch.equal(new, want)


@gpu
def test_weight_written_just_before_its_use(cuda_device):
    # the projection is launched as a dependent of the kernels that write its operands
    for seed in range(5):
        for rows in (2, 64, 400):
            h, w = inputs(cuda_device, rows, 512, 2048, seed=seed)
            torch.cuda.synchronize()
            weight = Int8Weight.from_weight(w)
            out = lm_head_logits_int8(h, weight.q, weight.scale)
            torch.cuda.synchronize()
            assert torch.equal(out, lm_head_logits_int8(h, weight.q, weight.scale))


@gpu
def test_head_sampler_and_scores_as_one_step(cuda_device):
    # hidden states -> 8-bit projection -> CFG chain and draw -> scores of the drawn tokens
    pairs, d, vocab = 64, 768, 4096
    h, w = inputs(cuda_device, 2 * pairs, d, vocab, seed=35)
    weight = Int8Weight.from_weight(w * 5)
    u = torch.rand(pairs, device=cuda_device)

    def make(**kw):
        return S.FusedSampler(vocab_size=vocab, num_rows=pairs, device=cuda_device, cfg_scale=1.5, time_shift_range=(0, 2000),
                              temperature=0.9, top_p=0.9, **kw)

    a, b = make(token_logprobs=5), make(return_scores=True)
    ids_a = a.step_hidden(h, weight, uniforms=u).clone()
    logits = lm_head_logits_int8(h, weight.q, weight.scale)
    ids_b = b.step(logits, uniforms=u).clone()
    assert torch.equal(a.lm_logits, logits) and torch.equal(ids_a, ids_b) and torch.equal(a.mono_state, b.mono_state)
    want = token_logprobs(b.scores, ids_b, top_n=5)
    for x, y in zip(a.token_logprobs, want):
        assert torch.equal(x, y)
    assert bool((a.token_logprobs.logprobs <= 0).all())
    # the same step captured and replayed
    c = make(token_logprobs=5)
    graph = torch.cuda.CUDAGraph()
    state = c.mono_state.clone()
    with torch.cuda.graph(graph):
        c.step_hidden(h, weight, uniforms=u)
    c.mono_state.copy_(state)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out_ids, ids_a) and torch.equal(c.token_logprobs.logprobs, want.logprobs)
    with pytest.raises(ValueError):
        a.step_hidden(h[:10], weight, uniforms=u)
    with pytest.raises(ValueError):
        a.step_hidden(h, Int8Weight(weight.q[:4000], weight.scale[:4000]), uniforms=u)


@gpu
def test_training_through_the_bf16_head(cuda_device):
    # the bf16 projection's logits, scored, and the gradient carried back to the hidden states by the product with the weight
    h, w = inputs(cuda_device, 96, 256, 1000, seed=12)
    wb = w.to(torch.bfloat16)
    logits = S.lm_head_logits(h, wb).requires_grad_(True)
    tokens = torch.randint(0, 1000, (96,), device=cuda_device)
    r = token_logprobs(logits, tokens)
    (-(r.logprobs.mean()) - 0.01 * r.entropy.mean() + 1e-3 * r.lse.square().mean()).backward()
    x = logits.detach().double().requires_grad_(True)
    logp = torch.log_softmax(x, 1)
    loss = -logp.gather(1, tokens[:, None]).mean() + 0.01 * (logp.exp() * logp).sum(1).mean() + 1e-3 * torch.logsumexp(x, 1).square().mean()
    loss.backward()
    # one bf16 rounding (2^-8 relative) plus fp32 noise far below it
    assert float(((logits.grad.double() - x.grad).abs() - 2.0 ** -8 * x.grad.abs() - 1e-9).max()) <= 0


# ------------------------------------------------------------------ rows whose scale is a small subnormal


def subnormal_rows(cols, seed):
    """fp32 rows whose largest magnitudes are a few thousand steps of 2^-149 at most: their scales keep few bits,
    so that quotients of up to 190 come out before they are held to 127."""
    tops = torch.tensor([1, 63, 64, 100, 127, 150, 190, 191, 318, 6000, 12000, 16000, 16129, 30000])
    g = torch.Generator().manual_seed(seed)
    steps = (torch.rand((len(tops), cols), generator=g) * (tops[:, None] + 1)).to(torch.int32)
    steps[:, 0] = steps[:, 1] = tops.to(torch.int32)
    negative = torch.rand((len(tops), cols), generator=g) < 0.5
    negative[:, 0], negative[:, 1] = False, True
    return torch.where(negative, steps | torch.tensor(-2 ** 31, dtype=torch.int32), steps).view(torch.float32)


def held_quantize(x):
    scale = x.abs().amax(1) * torch.tensor(1 / 127, dtype=torch.float32)
    q = torch.where((scale > 0)[:, None], x / scale[:, None], 0.0)
    return torch.round(q).clamp(-127, 127).to(torch.int8), scale


def test_quotients_of_subnormal_scales_pass_127():
    x = subnormal_rows(40, 0)
    scale = x.abs().amax(1) * torch.tensor(1 / 127, dtype=torch.float32)
    assert float((x / scale[:, None])[scale > 0].max()) == 190.0  # what the kernels must not store as -66


@gpu
@pytest.mark.parametrize("cols", [40, 33, 1000, 5001])
def test_quantize_rows_of_subnormal_scales(cuda_device, cols):
    x = subnormal_rows(cols, cols)
    q, scale = quantize_rows(x.to(cuda_device))
    want_q, want_s = held_quantize(x)
    same(scale, want_s)
    same(q, want_q)


@gpu
@pytest.mark.parametrize("rows", [7, 140])
@pytest.mark.parametrize("cols", [40, 33])
def test_logits_of_subnormal_scales(cuda_device, rows, cols):
    x = subnormal_rows(cols, cols)[4:11].repeat(rows // 7, 1)
    g = torch.Generator().manual_seed(1)
    wide = torch.zeros((50, 48), dtype=torch.int8)
    wide[:, :cols] = torch.randint(-128, 128, (50, cols), generator=g).to(torch.int8)
    ws = torch.full((50,), 2.0 ** 120)
    wide_d = wide.to(cuda_device)
    out = lm_head_logits_int8(x.to(cuda_device), wide_d[:, :cols], ws.to(cuda_device), out_dtype=torch.float32)
    q, scale = held_quantize(x)
    same(out, plain_logits(q, scale, wide[:, :cols], ws, torch.float32))


# ------------------------------------------------------------------ the largest row count


@gpu
def test_quantize_as_many_rows_as_the_count_holds(cuda_device):
    rows = 2 ** 31 - 1
    x = torch.full((rows,), 3.0, dtype=torch.bfloat16, device=cuda_device)
    x[-1], x[-2] = -3.0, 0.0
    q = torch.zeros(rows, dtype=torch.int8, device=cuda_device)
    scale = torch.empty(rows, device=cuda_device)
    a = N.sized(N.MtrQuantizeArgs, x=x.data_ptr(), x_row_stride=1, x_dtype=N.DTYPE_BF16, rows=rows, cols=1, q=q.data_ptr(),
                q_row_stride=1, scale=scale.data_ptr())
    N.quantize_rows_launch(a, torch.cuda.current_stream().cuda_stream)
    want = float(torch.tensor(3.0) * torch.tensor(1 / 127, dtype=torch.float32))
    assert q[-1] == -127 and q[-2] == 0 and scale[-2] == 0 and scale[-1] == want
    assert bool((q[:-2] == 127).all()) and bool((scale[:-2] == want).all())


# ------------------------------------------------------------------ matrices side by side in one buffer


@pytest.mark.parametrize("at,code", [(100, N.OK), (99, N.ERR_BAD_PARAM), (300 - 77, N.OK), (300 - 76, N.ERR_BAD_PARAM),
                                     (300 + 100, N.OK), (-77, N.OK), (-76, N.ERR_BAD_PARAM), (0, N.ERR_BAD_PARAM)])
def test_hidden_and_logits_may_share_a_buffer_of_wider_rows(at, code):
    a = _proj_args()
    a.hidden_row_stride = a.logits_row_stride = 300
    a.logits = a.hidden + 2 * at
    lib = N.load()
    assert lib.mtr_lmhead_i8_validate(ctypes.byref(a)) == code
    a.logits_row_stride = 301  # rows that drift against each other may meet
    assert lib.mtr_lmhead_i8_validate(ctypes.byref(a)) == N.ERR_BAD_PARAM


@pytest.mark.parametrize("at,code", [(128, N.OK), (127, N.ERR_BAD_PARAM), (256 - 64, N.OK), (256 - 63, N.ERR_BAD_PARAM)])
def test_rows_and_their_int8_may_share_a_buffer_of_wider_rows(at, code):
    a = _quant_args(x_row_stride=128, q_row_stride=256)
    a.q = a.x + at
    assert N.load().mtr_quantize_rows_validate(ctypes.byref(a)) == code


@gpu
@pytest.mark.parametrize("rows", [3, 150])
def test_hidden_and_logits_in_one_buffer(cuda_device, rows):
    h, w = inputs(cuda_device, rows, 200, 301, seed=21)
    weight = Int8Weight.from_weight(w)
    both = torch.full((rows, 520), 7.0, dtype=torch.bfloat16, device=cuda_device)
    both[:, :200] = h
    lm_head_logits_int8(both[:, :200], weight.q, weight.scale, both[:, 204:505])
    assert torch.equal(both[:, 204:505], lm_head_logits_int8(h, weight.q, weight.scale))
    assert torch.equal(both[:, :200], h) and bool((both[:, 200:204] == 7.0).all()) and bool((both[:, 505:] == 7.0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantized_weight(cuda_device, dtype):
    _, w = inputs(cuda_device, 1, 203, 37, seed=30)
    w[4] = 0.0
    w = w.to(dtype)
    back = Int8Weight.from_weight(w).dequantize()
    assert back.shape == w.shape and back.dtype == torch.float32 and bool((back[4] == 0).all())
    # half a step of the row's scale, and the roundings of the scale, the quotient and the product
    step = w.float().abs().amax(1, keepdim=True) / 127
    assert bool(((back - w.float()).abs() <= 0.5 * step + 4 * 2.0 ** -24 * 127 * step).all())
