"""Bounded waits of the tensor-core projections that give up: what was not
computed reads NaN, the wait is counted for the device and in the caller's word,
the sampler pads the rows, and the next call is as if nothing had happened.  The
test hook makes the epilogues take their first wait as run out; where a CTA has
more tiles than two, the waits of the other roles run out by themselves (200 ms)."""

import ctypes
import math

import pytest
import torch

from mapperatorinator_b200 import _native as N
from mapperatorinator_b200 import sampling as S
from mapperatorinator_b200.int8_head import Int8Weight, lm_head_logits_int8, lmhead_i8_args

gpu = pytest.mark.gpu


def test_count_argument_is_checked_on_the_host():
    lib = N.load()
    assert lib.mtr_projection_timeouts(None, None) == N.ERR_NULL_ARG
    lib.mtr_projection_test_waits(1)
    lib.mtr_projection_test_waits(0)


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


def _inputs(device, rows, d, vocab, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    h = torch.randn((rows, d), generator=g, device=device).to(torch.bfloat16)
    w = torch.randn((vocab, d), generator=g, device=device) * 0.02
    return h, w


@gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("rows,d,vocab", [(140, 200, 300), (9, 64, 77), (128, 300, 16384), (128, 64, 65536), (512, 4096, 16384)])
def test_int8_projection_that_gives_up(cuda_device, giving_up, out_dtype, rows, d, vocab):
    h, w = _inputs(cuda_device, rows, d, vocab)
    weight = Int8Weight.from_weight(w)
    want = lm_head_logits_int8(h, weight.q, weight.scale, out_dtype=out_dtype)
    before = S.projection_timeouts(cuda_device)
    wide = torch.full((rows + 1, vocab + 5), 7.0, dtype=out_dtype, device=cuda_device)
    out = wide[:rows, :vocab]
    with giving_up:
        lm_head_logits_int8(h, weight.q, weight.scale, out)
    assert bool(torch.isnan(out).all())
    assert bool((wide[rows:] == 7.0).all()) and bool((wide[:, vocab:] == 7.0).all())
    count = S.projection_timeouts()
    assert count > before
    lm_head_logits_int8(h, weight.q, weight.scale, out)
    assert torch.equal(out, want) and S.projection_timeouts() == count


@gpu
@pytest.mark.parametrize("rows,d,vocab", [(128, 64, 131072), (1024, 768, 32768)])
def test_waits_that_run_out(cuda_device, giving_up, rows, d, vocab):
    # more than two tiles a CTA (a pair): the products wait for an accumulator that no epilogue frees, the loads for a stage
    h, w = _inputs(cuda_device, rows, d, vocab)
    weight = Int8Weight.from_weight(w)
    out = torch.full((rows, vocab), 7.0, dtype=torch.bfloat16, device=cuda_device)
    word = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    a, work = lmhead_i8_args(h, weight.q, weight.scale, out)
    a.error_word = word.data_ptr()
    with giving_up:
        N.lmhead_i8_launch(a, torch.cuda.current_stream().cuda_stream)
    assert bool(torch.isnan(out).all())
    assert word.item() & 6 == 6 and word.item() & ~7 == 0  # the epilogue's and the products', perhaps the loads'
    word.zero_()
    N.lmhead_i8_launch(a, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, lm_head_logits_int8(h, weight.q, weight.scale)) and word.item() == 0
    del work


@gpu
@pytest.mark.parametrize("rows,d,vocab,tile_n", [(130, 128, 520, 0), (256, 768, 4096, 64), (256, 768, 4096, 128)])
def test_bf16_projection_that_gives_up(cuda_device, giving_up, rows, d, vocab, tile_n):
    h, w = _inputs(cuda_device, rows, d, vocab)
    w = w.to(torch.bfloat16)
    want = S.lm_head_logits(h, w, tile_n=tile_n)
    before = S.projection_timeouts(cuda_device)
    wide = torch.full((rows + 1, vocab + 8), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = wide[:rows, :vocab]
    with giving_up:
        S.lm_head_logits(h, w, out, tile_n=tile_n)
    assert bool(torch.isnan(out).all())
    assert bool((wide[rows:] == 7.0).all()) and bool((wide[:, vocab:] == 7.0).all())
    count = S.projection_timeouts()
    assert count > before
    S.lm_head_logits(h, w, out, tile_n=tile_n)
    assert torch.equal(out, want) and S.projection_timeouts() == count


@gpu
@pytest.mark.parametrize("int8", [True, False])
def test_a_step_whose_projection_gives_up(cuda_device, giving_up, int8):
    pairs, d, vocab, pad = 32, 256, 1024, 3
    h, w = _inputs(cuda_device, 2 * pairs, d, vocab)
    weight = Int8Weight.from_weight(w) if int8 else w.to(torch.bfloat16)
    u = torch.rand(pairs, device=cuda_device)
    sampler = S.FusedSampler(vocab_size=vocab, num_rows=pairs, device=cuda_device, cfg_scale=1.5, pad_token_id=pad, token_logprobs=2)
    want = sampler.step_hidden(h, weight, uniforms=u).clone()
    assert S.row_status_report(sampler.status)["padded"] == []
    with giving_up:
        ids = sampler.step_hidden(h, weight, uniforms=u)
    report = S.row_status_report(sampler.status, ids, pad)
    assert report["nonfinite"] == report["padded"] == list(range(pairs))
    assert bool((ids == pad).all()) and all(math.isnan(v) for v in sampler.token_logprobs.logprobs.tolist())
    assert torch.equal(sampler.step_hidden(h, weight, uniforms=u), want)


@gpu
def test_count_is_not_read_while_capturing(cuda_device):
    S.projection_timeouts(cuda_device)
    x = torch.zeros(4, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(N.SamplerError):
            S.projection_timeouts(cuda_device)
    graph.replay()
    n = ctypes.c_uint32(7)
    assert N.load().mtr_projection_timeouts(ctypes.byref(n), None) == N.OK and n.value == S.projection_timeouts(cuda_device)
    assert bool((x == 1).all())
