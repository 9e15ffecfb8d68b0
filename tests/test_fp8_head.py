"""The output projection in 8-bit floating point.  The quantisation is defined to the
bit (fp32 quotients, one rounding to e4m3) and compared for equality.  The logits
are compared with float64 sums of the quantised values: a block's products are
exact in fp32, and its 128 terms are added in fp32 in some order, rounded or cut
off, within 128 2^-23 of the sum of their magnitudes; each of the n blocks is scaled
(two roundings) and added (one), so with M = sum |h w|
    |error| <= (128 2^-23 + (n + 3) 2^-24) M + eps / 2 |logit|."""

import ctypes
import math

import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.fp8_head import Fp8Weight, lm_head_logits_fp8, lmhead_f8_args, quantize_blocks
from mapperatorinator_b200.scoring import token_logprobs
from mapperatorinator_b200.speculative import verify_drafts
from mapperatorinator_b200.distillation import distillation_loss_and_grad

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain_quantize(x, block_rows):
    x = x.float().cpu()
    rows, cols = x.shape
    high, wide = -(-rows // block_rows), -(-cols // 128)
    padded = torch.zeros((high * block_rows, wide * 128))
    padded[:rows, :cols] = x
    cube = padded.view(high, block_rows, wide, 128)
    top = cube.abs().amax(dim=(1, 3))
    bad = ~torch.isfinite(cube).all(dim=3).all(dim=1)
    scale = torch.where(bad, math.nan, top * torch.tensor(1 / 448, dtype=torch.float32))
    each = scale[:, None, :, None]
    q = torch.where(each > 0, cube / each, 0.0).nan_to_num(0.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.view(high * block_rows, wide * 128)[:rows, :cols], scale


def dequantize(q, scale, block_rows):
    rows, cols = q.shape
    return q.double() * scale.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def inputs(device, rows, d, vocab, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    h = torch.randn((rows, d), generator=g, device=device)
    h[:, ::97] *= 20.0  # large channels
    w = torch.randn((vocab, d), generator=g, device=device) * 0.02
    return h.to(dtype), w


def check(out, h, weight):
    """Against float64 sums of the quantised hidden states (which are checked by themselves)."""
    q, scale = quantize_blocks(h)
    a, b = dequantize(q, scale, 1), dequantize(weight.q, weight.scale, 128)
    want, size = a @ b.T, a.abs() @ b.abs().T
    n = scale.shape[1]
    tol = (128 * 2.0 ** -23 + (n + 3) * 2.0 ** -24) * size + (torch.finfo(out.dtype).eps / 2) * (want.abs() + 2.0 ** -16 * size) \
        + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(out), nan)
    err = torch.where(nan, 0.0, (out.double() - want).abs() - tol)
    assert float(err.max()) <= 0, float(err.max())


def same(got, want):
    got, want = got.cpu(), want.cpu()
    assert got.dtype == want.dtype and got.shape == want.shape
    got, want = got.float(), want.float()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan]), int((got[~nan] != want[~nan]).sum())


# ------------------------------------------------------------------ CPU


def _quant_args():
    return N.sized(N.MtrQuantizeBlocksArgs, x=0x100000, x_row_stride=200, x_dtype=N.DTYPE_BF16, rows=4, cols=200, block_rows=1, q=0x200000,
                   q_row_stride=208, scale=0x300000, scale_row_stride=2)


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0, x=None), N.OK), (dict(block_rows=128), N.OK), (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(cols=0), N.ERR_BAD_SHAPE),
    (dict(rows=N.MAX_F8_ROWS + 1), N.ERR_BAD_SHAPE), (dict(cols=N.MAX_F8_D_MODEL + 1), N.ERR_BAD_SHAPE), (dict(block_rows=2), N.ERR_BAD_PARAM),
    (dict(x_row_stride=199), N.ERR_BAD_SHAPE), (dict(q_row_stride=196), N.ERR_BAD_SHAPE), (dict(scale_row_stride=1), N.ERR_BAD_SHAPE),
    (dict(x_dtype=3), N.ERR_BAD_PARAM), (dict(q=None), N.ERR_NULL_ARG), (dict(scale=None), N.ERR_NULL_ARG), (dict(x=0x100001), N.ERR_ALIGNMENT),
    (dict(q=0x200002), N.ERR_ALIGNMENT), (dict(q_row_stride=206), N.ERR_ALIGNMENT), (dict(scale=0x300002), N.ERR_ALIGNMENT),
    (dict(q=0x100010), N.ERR_BAD_PARAM), (dict(scale=0x200010), N.ERR_BAD_PARAM), (dict(struct_size=1), N.ERR_ABI)])
def test_quantize_arguments_are_checked_on_the_host(kw, code):
    a = _quant_args()
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_quantize_blocks_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_quantize_blocks_launch(ctypes.byref(a), None) == code


def _proj_args():
    return N.sized(N.MtrLmHeadF8Args, hidden=0x1000000, hidden_row_stride=200, weight=0x2000000, weight_row_stride=208,
                   weight_scale=0x3000000, scale_row_stride=2, logits=0x4000000, logits_row_stride=300, hidden_dtype=N.DTYPE_BF16,
                   logits_dtype=N.DTYPE_BF16, rows=900, d_model=200, vocab=300, workspace=0x5000000, workspace_bytes=1 << 20)


@pytest.mark.parametrize("kw,code", [
    ({}, N.OK), (dict(rows=0, hidden=None), N.OK), (dict(rows=-1), N.ERR_BAD_SHAPE), (dict(rows=N.MAX_F8_ROWS + 1), N.ERR_BAD_SHAPE),
    (dict(d_model=0), N.ERR_BAD_SHAPE), (dict(d_model=N.MAX_F8_D_MODEL + 1), N.ERR_BAD_SHAPE), (dict(vocab=0), N.ERR_BAD_SHAPE),
    (dict(vocab=N.MAX_VOCAB + 1), N.ERR_BAD_SHAPE), (dict(hidden_dtype=3), N.ERR_BAD_PARAM), (dict(logits_dtype=-1), N.ERR_BAD_PARAM),
    (dict(weight=None), N.ERR_NULL_ARG), (dict(weight_scale=None), N.ERR_NULL_ARG), (dict(workspace=None), N.ERR_NULL_ARG),
    (dict(workspace_bytes=900 * 208), N.ERR_BAD_SHAPE), (dict(rows=8, workspace=None, workspace_bytes=0), N.OK),
    (dict(workspace=0x5000010), N.ERR_ALIGNMENT), (dict(weight_row_stride=216), N.ERR_ALIGNMENT), (dict(weight=0x2000008), N.ERR_ALIGNMENT),
    (dict(weight_row_stride=192), N.ERR_BAD_SHAPE), (dict(logits_row_stride=299), N.ERR_BAD_SHAPE), (dict(scale_row_stride=1), N.ERR_BAD_SHAPE),
    (dict(hidden_row_stride=199), N.ERR_BAD_SHAPE), (dict(logits=0x1000000), N.ERR_BAD_PARAM), (dict(weight_scale=0x4000000), N.ERR_BAD_PARAM),
    (dict(workspace=0x4000000), N.ERR_BAD_PARAM), (dict(error_word=2), N.ERR_ALIGNMENT), (dict(abi_version=9), N.ERR_ABI)])
def test_projection_arguments_are_checked_on_the_host(kw, code):
    a = _proj_args()
    for k, v in kw.items():
        setattr(a, k, v)
    lib = N.load()
    assert lib.mtr_lmhead_f8_validate(ctypes.byref(a)) == code
    if code != N.OK or a.rows == 0:
        assert lib.mtr_lmhead_f8_launch(ctypes.byref(a), None) == code


def test_projection_and_sampler_must_share_the_logits():
    lm, a = _proj_args(), N.new_args()
    a.logits, a.logits_row_stride, a.logits_dtype, a.vocab, a.num_rows = lm.logits, 300, N.DTYPE_BF16, 300, 900
    a.select_mode, a.out_ids = N.SELECT_ARGMAX, 0x6000000
    lib = N.load()
    for field, value, code in (("logits", 0x7000000, N.ERR_BAD_PARAM), ("logits_row_stride", 301, N.ERR_BAD_PARAM),
                               ("logits_dtype", N.DTYPE_F16, N.ERR_BAD_PARAM), ("num_rows", 901, N.ERR_BAD_SHAPE)):
        b = N.MtrSamplerArgs()
        ctypes.pointer(b)[0] = a
        setattr(b, field, value)
        assert lib.mtr_lmhead_f8_sample_launch(ctypes.byref(lm), ctypes.byref(b), None) == code, field
    lm.rows = a.num_rows = 0
    assert lib.mtr_lmhead_f8_sample_launch(ctypes.byref(lm), ctypes.byref(a), None) == N.OK


def test_workspace_sizes():
    assert N.lmhead_f8_workspace(0, 64, 100) == 0 and N.lmhead_f8_workspace(4, 0, 100) == 0
    assert N.lmhead_f8_workspace(3, 100, 4096) == 0  # few rows
    assert N.lmhead_f8_workspace(301, 200, 77) == 62720 + 304 * 8  # 301 rows of 208 bytes, the scales of 304 on the next 256-byte boundary
    assert N.lmhead_f8_workspace(N.MAX_F8_ROWS, N.MAX_F8_D_MODEL, 1) == (1 << 39) + (1 << 34)


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 16))
    with pytest.raises(ValueError):
        quantize_blocks(x)
    with pytest.raises(ValueError):
        lm_head_logits_fp8(x, x.to(torch.float8_e4m3fn), torch.ones((1, 1)))


# ------------------------------------------------------------------ GPU

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 128), (130, 129), (256, 768), (17, 1001), (2, 4096), (3, 70001)])
def test_quantize_blocks(cuda_device, dtype, block_rows, rows, cols):
    x, _ = inputs(cuda_device, rows, cols, 1, dtype, seed=rows + cols)
    q, scale = quantize_blocks(x, block_rows=block_rows)
    want_q, want_s = plain_quantize(x, block_rows)
    same(scale, want_s)
    same(q, want_q)
    assert q.stride(0) % 16 == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [40, 1000])
def test_quantize_odd_blocks(cuda_device, dtype, block_rows, cols):
    x, _ = inputs(cuda_device, 10, cols, 1, dtype, seed=3)
    x[0] = 0.0
    x[1, 7] = math.nan
    x[2, 8] = math.inf
    x[3, cols - 1] = -math.inf
    x[4] = torch.finfo(dtype).max
    x[5] = x[5] * torch.finfo(dtype).tiny  # subnormal scales, or none
    x[6] = torch.finfo(dtype).tiny * 0.25 if dtype == torch.float32 else torch.finfo(dtype).smallest_normal
    x[7] = (torch.arange(cols, device=cuda_device) % 97 - 48 + 0.5).to(dtype)  # halves of e4m3's steps
    x[7, ::128] = 448.0
    x[8] = 0.0
    x[8, cols - 1] = -3.0
    if block_rows > 1:
        for r in range(10):  # a row at a time decides the block
            y = torch.zeros_like(x)
            y[r] = x[r]
            q, scale = quantize_blocks(y, block_rows=128)
            want_q, want_s = plain_quantize(y, 128)
            same(scale, want_s)
            same(q, want_q)
    q, scale = quantize_blocks(x, block_rows=block_rows)
    want_q, want_s = plain_quantize(x, block_rows)
    same(scale, want_s)
    same(q, want_q)


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_strided_rows(cuda_device, block_rows):
    x, _ = inputs(cuda_device, 9, 203, 1, torch.float16, seed=5)
    wide = torch.full((9, 211), math.nan, dtype=torch.float16, device=cuda_device)
    wide[:, 3:206] = x
    q, scale = quantize_blocks(wide[:, 3:206], block_rows=block_rows)
    want_q, want_s = plain_quantize(x, block_rows)
    same(q, want_q)
    same(scale, want_s)
    assert quantize_blocks(x[:0], block_rows=block_rows)[0].shape == (0, 203)
    assert Fp8Weight.from_weight(x).dequantize().shape == (9, 203)


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("rows,d,vocab,dtype", [
    (1, 1, 1, torch.float32), (1, 16, 8, torch.bfloat16), (8, 2048, 1000, torch.bfloat16), (5, 1001, 300, torch.float16), (2, 768, 4096, torch.bfloat16),
    (8, 100, 131072, torch.float32), (1, 8192, 77, torch.bfloat16), (1, 8193, 77, torch.bfloat16), (9, 64, 20000, torch.float32),
    (3, 15, 3, torch.bfloat16), (4, 2048, 16000, torch.float32), (7, 1500, 40000, torch.bfloat16), (2, 129, 15, torch.float16),
    (128, 768, 4096, torch.bfloat16), (33, 100, 77, torch.float16), (129, 1001, 4099, torch.float16), (300, 64, 520, torch.float32),
    (256, 128, 8192, torch.bfloat16), (513, 2048, 1000, torch.bfloat16), (1030, 96, 264, torch.float32), (64, 3000, 131072, torch.bfloat16),
    (300, 2100, 8200, torch.bfloat16), (300, 64, 40000, torch.bfloat16), (600, 640, 20000, torch.float16), (2000, 4100, 5000, torch.bfloat16)])
def test_logits(cuda_device, out_dtype, rows, d, vocab, dtype):
    h, w = inputs(cuda_device, rows, d, vocab, dtype, seed=rows + d + vocab)
    weight = Fp8Weight.from_weight(w)
    out = lm_head_logits_fp8(h, weight.q, weight.scale, out_dtype=out_dtype)
    check(out, h, weight)
    assert torch.equal(out, lm_head_logits_fp8(h, weight.q, weight.scale, out_dtype=out_dtype))


@gpu
@pytest.mark.parametrize("rows", [7, 147])
def test_odd_rows_and_weights(cuda_device, rows):
    h, w = inputs(cuda_device, 7, 300, 300, torch.bfloat16, seed=2)
    h[1], h[2, 5], h[3, 299] = 0.0, math.nan, math.inf
    w[:128, :128] = 0.0
    w[130, 290] = math.nan  # 128 ids whose scale is NaN
    h = torch.cat([h] * (rows // 7))
    weight = Fp8Weight.from_weight(w)
    out = lm_head_logits_fp8(h, weight.q, weight.scale)
    check(out, h, weight)
    assert bool(torch.isnan(out[2:4]).all()) and bool(torch.isnan(out[:, 128:256]).all()) and bool((out[1, :128] == 0).all())


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("vocab,stride,offset", [(300, 301, 1), (256, 260, 0), (4096, 4104, 8), (4099, 4100, 2), (4099, 4104, 0),
                                                 (29, 32, 8), (4102, 4104, 0), (3, 8, 0)])
def test_strides_and_what_lies_behind(cuda_device, out_dtype, vocab, stride, offset):
    rows, d = 140, 200
    h, w = inputs(cuda_device, rows, d, vocab, seed=6)
    wide_h = torch.full((rows, 300), math.nan, dtype=torch.bfloat16, device=cuda_device)
    wide_h[:, 51:251] = h
    weight = Fp8Weight.from_weight(w)
    wide_w = torch.full((vocab, 256), math.nan, device=cuda_device).to(torch.float8_e4m3fn)
    wide_w[:, :d] = weight.q
    wide_s = torch.full((weight.scale.shape[0], 5), math.nan, device=cuda_device)
    wide_s[:, 1:3] = weight.scale
    buf = torch.full((offset + (rows + 3) * stride,), 7.0, dtype=out_dtype, device=cuda_device)
    out = buf[offset:].as_strided((rows, vocab), (stride, 1))
    got = lm_head_logits_fp8(wide_h[:, 51:251], wide_w[:, :d], wide_s[:, 1:3], out)
    assert got is out
    assert torch.equal(out, lm_head_logits_fp8(h, weight.q, weight.scale, out_dtype=out_dtype))
    few_buf = torch.full((offset + 9 * stride,), 7.0, dtype=out_dtype, device=cuda_device)
    few = few_buf[offset:].as_strided((7, vocab), (stride, 1))
    lm_head_logits_fp8(wide_h[:7, 51:251], wide_w[:, :d], wide_s[:, 1:3], few)  # few rows: another kernel
    check(few, h[:7], weight)
    rest = torch.ones_like(few_buf, dtype=torch.bool)
    rest[offset:].as_strided((7, vocab), (stride, 1)).fill_(False)
    assert bool((few_buf[rest] == 7.0).all())
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[offset:].as_strided((rows, vocab), (stride, 1)).fill_(False)
    assert bool((buf[rest] == 7.0).all())  # columns behind the vocabulary and rows behind the last


@gpu
def test_refusals(cuda_device):
    h, w = inputs(cuda_device, 4, 64, 80)
    q, s = Fp8Weight.from_weight(w)
    odd = torch.zeros((80, 65), device=cuda_device).to(torch.float8_e4m3fn)[:, :64]
    for bad, exc in ((lambda: lm_head_logits_fp8(h[:, :32], q, s), ValueError), (lambda: lm_head_logits_fp8(h.double(), q, s), TypeError),
                     (lambda: lm_head_logits_fp8(h, q.float(), s), TypeError), (lambda: lm_head_logits_fp8(h, q, s[:0]), ValueError),
                     (lambda: lm_head_logits_fp8(h, q, s.double()), TypeError), (lambda: lm_head_logits_fp8(h, odd, s), ValueError),
                     (lambda: lm_head_logits_fp8(h, q, s.cpu()), ValueError), (lambda: lm_head_logits_fp8(h.T, q, s), ValueError),
                     (lambda: lm_head_logits_fp8(h, q, s[0]), ValueError), (lambda: lm_head_logits_fp8(h, q, s, h), ValueError),
                     (lambda: lm_head_logits_fp8(h, q, s, out_dtype=torch.int32), TypeError),
                     (lambda: quantize_blocks(h[:, :0]), ValueError), (lambda: quantize_blocks(h.long()), TypeError),
                     (lambda: quantize_blocks(h, block_rows=64), ValueError)):
        with pytest.raises(exc):
            bad()
    assert lm_head_logits_fp8(h[:0], q, s).shape == (0, 80)


@gpu
@pytest.mark.parametrize("rows", [2, 130])
def test_streams_and_graphs(cuda_device, rows):
    h, w = inputs(cuda_device, 130, 768, 1000, seed=9)
    weight = Fp8Weight.from_weight(w)
    call = lambda: lm_head_logits_fp8(h[:rows], weight.q, weight.scale)  # noqa: E731
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
    want = call()
    for graph, _ in graphs * 2:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs)


@gpu
def test_weight_written_just_before_its_use(cuda_device):
    # the projection is launched as a dependent of the kernels that write its operands
    for seed in range(5):
        for rows in (2, 64, 400):
            h, w = inputs(cuda_device, rows, 512, 2048, seed=seed)
            torch.cuda.synchronize()
            weight = Fp8Weight.from_weight(w)
            out = lm_head_logits_fp8(h, weight.q, weight.scale)
            torch.cuda.synchronize()
            assert torch.equal(out, lm_head_logits_fp8(h, weight.q, weight.scale))


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("d,vocab", [(128, 16), (768, 4097), (1001, 8192), (6000, 40), (385, 70001), (2900, 8192)])
def test_few_rows(cuda_device, rows, d, vocab):
    h, w = inputs(cuda_device, 8, d, vocab, seed=rows + d)
    weight = Fp8Weight.from_weight(w)
    out = lm_head_logits_fp8(h[:rows], weight.q, weight.scale, out_dtype=torch.float32)
    check(out, h[:rows], weight)
    alone = torch.cat([lm_head_logits_fp8(h[r:r + 1], weight.q, weight.scale, out_dtype=torch.float32) for r in range(rows)])
    check(alone, h[:rows], weight)


@gpu
@pytest.mark.parametrize("pairs", [1, 40])
def test_sampler_takes_the_weight(cuda_device, pairs):
    d, vocab = 320, 1000
    h, w = inputs(cuda_device, 2 * pairs, d, vocab, seed=4)
    weight = Fp8Weight.from_weight(w)
    u = torch.rand(pairs, device=cuda_device)
    make = lambda: S.FusedSampler(vocab_size=vocab, num_rows=pairs, device=cuda_device, cfg_scale=1.5, top_k=20, token_logprobs=3)  # noqa: E731
    a, b = make(), make()
    ids = a.step_hidden(h, weight, uniforms=u).clone()
    logits = lm_head_logits_fp8(h, weight.q, weight.scale)
    assert torch.equal(a.lm_logits, logits)
    assert torch.equal(b.step(logits, uniforms=u), ids)
    assert torch.equal(a.token_logprobs.logprobs, b.token_logprobs.logprobs)


@pytest.fixture
def giving_up(cuda_device):
    N.load()

    class Switch:
        def __enter__(self):
            N.projection_test_waits(True)

        def __exit__(self, *exc):
            N.projection_test_waits(False)

    yield Switch()
    N.projection_test_waits(False)


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("rows,d,vocab", [(140, 200, 300), (9, 64, 77), (128, 300, 16384), (128, 64, 65536), (512, 4096, 16384)])
def test_projection_that_gives_up(cuda_device, giving_up, out_dtype, rows, d, vocab):
    h, w = inputs(cuda_device, rows, d, vocab)
    weight = Fp8Weight.from_weight(w)
    want = lm_head_logits_fp8(h, weight.q, weight.scale, out_dtype=out_dtype)
    before = S.projection_timeouts(cuda_device)
    wide = torch.full((rows + 1, vocab + 5), 7.0, dtype=out_dtype, device=cuda_device)
    out = wide[:rows, :vocab]
    word = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    a, work = lmhead_f8_args(h, weight.q, weight.scale, out)
    a.error_word = word.data_ptr()
    with giving_up:
        N.lmhead_f8_launch(a, torch.cuda.current_stream().cuda_stream)
    assert bool(torch.isnan(out).all())
    assert bool((wide[rows:] == 7.0).all()) and bool((wide[:, vocab:] == 7.0).all())
    assert word.item() & 4 and word.item() & ~7 == 0
    count = S.projection_timeouts()
    assert count > before
    lm_head_logits_fp8(h, weight.q, weight.scale, out)
    assert torch.equal(out, want) and S.projection_timeouts() == count
    del work


@gpu
def test_a_draft_model_beside_the_target(cuda_device):
    """The operators as they are used together: the target's head scores a prefix and the drafts of each sequence, the
    draft's tokens are verified, and the draft's head learns from the target's alternatives at the same positions."""
    batch, drafts, d, small, vocab = 12, 4, 512, 128, 2000
    g = torch.Generator(device=cuda_device).manual_seed(7)
    positions = torch.randn((batch * (drafts + 1), d), generator=g, device=cuda_device, dtype=torch.bfloat16)
    target = Fp8Weight.from_weight(torch.randn((vocab, d), generator=g, device=cuda_device) * 0.1)
    head = (torch.randn((vocab, small), generator=g, device=cuda_device) * 0.1).requires_grad_(True)
    squeeze = torch.randn((d, small), generator=g, device=cuda_device) * d ** -0.5
    hidden = positions.float() @ squeeze
    draft_logits = (hidden @ head.T).view(batch, drafts + 1, vocab)[:, :drafts]
    ids = torch.multinomial(torch.softmax(draft_logits.detach().reshape(-1, vocab), 1), 1, generator=g).view(batch, drafts)
    u = torch.rand((batch, drafts + 1), generator=g, device=cuda_device)

    logits = lm_head_logits_fp8(positions, target.q, target.scale, out_dtype=torch.float32)
    r = verify_drafts(logits.view(batch, drafts + 1, vocab), ids, draft_logits.detach(), uniforms=u)
    x = torch.log_softmax(logits.double(), 1).view(batch, drafts + 1, vocab)
    for b in range(batch):
        n = int(r.accepted[b])
        assert torch.equal(r.tokens[b, :n], ids[b, :n]) and 0 <= int(r.tokens[b, n]) < vocab and bool((r.tokens[b, n + 1:] == 0).all())
        for j in range(n + 1):
            assert abs(float(x[b, j, r.tokens[b, j]]) - float(r.logprobs[b, j])) < 1e-5  # fp32 sums of 2000 terms, logarithms of about 10
    teacher = token_logprobs(logits, top_n=32)
    student = hidden @ head.T
    loss, grad = distillation_loss_and_grad(student.detach(), teacher.top_ids, teacher.top_logprobs, tail=True)
    assert bool(torch.isfinite(loss).all()) and float(loss.detach().min()) >= 0
    from mapperatorinator_b200.distillation import distillation_loss
    (by_autograd,) = torch.autograd.grad(distillation_loss(student, teacher.top_ids, teacher.top_logprobs, tail=True).sum(), head)
    by_hand = grad.T @ hidden
    # 60 products of fp32 in two orders
    assert float((by_autograd - by_hand).abs().max()) <= 60 * 2.0 ** -23 * float((grad.abs().T @ hidden.abs()).max())


@gpu
@pytest.mark.parametrize("rows", [8, 127])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_sums_keep_24_bits(cuda_device, rows, sign):
    """Both kernels' instructions add products as fp32 does: 448 * 448 +- 2^-k, k to 6, has at most 24 bits, so a sum that
    keeps 24 of them is exact wherever in the block the small product stands; one rounding scales it."""
    h = torch.zeros((127, 128), device=cuda_device)
    h[:, 0] = 448.0
    h[torch.arange(127), torch.arange(127) + 1] = sign * 2.0 ** -3
    powers = torch.tensor([2.0 ** (3 - k) for k in range(-5, 7)], device=cuda_device)  # with 2^-3: 2^5 .. 2^-6
    w = powers[:, None].repeat(1, 128)
    w[:, 0] = 448.0
    q, one = w.to(torch.float8_e4m3fn), torch.ones((1, 1), device=cuda_device)
    assert torch.equal(q.float(), w)
    _, scale = quantize_blocks(h)
    exact = 448.0 * 448.0 + sign * 2.0 ** -3 * powers.double()
    want = (exact[None] * scale.double()).float()
    got = torch.cat([lm_head_logits_fp8(h[r:r + rows], q, one, out_dtype=torch.float32) for r in range(0, 127, rows)])
    assert got.shape == want.shape and torch.equal(got, want), (got != want).nonzero()[:5]
