"""A draft model's operators as a user calls them, beside their plain form in elementary torch operations.

  fp8      hidden states to logits through an output projection in 8-bit floating point: each row of hidden states is
           quantised in blocks of 128 values, the weight carries one scale for each 128 x 128 block
  distill  losses of a student's logits against a teacher's top ids, and the gradient of the logits
  verify   drafted tokens accepted or replaced under the target's distribution, from given random numbers
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 128
E4M3_MAX = 448.0
LEAST_REST = 2.0**-20  # a smaller rest of a teacher's mass is the rounding of the log probabilities that were given


def listed():
    return [
        # one song: the conditional and unconditional rows of a single step
        {"name": "fp8_song", "op": "fp8", "rows": 2, "d": 768, "vocab": 4096, "hidden": "bf16", "out": "bf16"},
        # odd sizes on every axis, half-precision hidden states, fp32 logits
        {"name": "fp8_ragged", "op": "fp8", "rows": 333, "d": 1001, "vocab": 4099, "hidden": "f16", "out": "f32"},
        # 64 sequences of four drafted tokens: five positions each, a wide vocabulary
        {"name": "fp8_drafts", "op": "fp8", "rows": 320, "d": 1024, "vocab": 65536, "hidden": "bf16", "out": "bf16"},
        # whole windows through a wide model, as a teacher reads them: bound by the tensor cores
        {"name": "fp8_large", "op": "fp8", "rows": 8192, "d": 4096, "vocab": 16384, "hidden": "bf16", "out": "bf16"},
        # a few positions of one song learned while it is served
        {"name": "distill_song", "op": "distill", "rows": 64, "vocab": 4096, "n": 5, "dtype": "f32", "tail": True, "train": True, "temperature": 1.0, "masked": 0.5},
        # a training step over windows, the teacher's best 20 renormalised
        {"name": "distill_windows", "op": "distill", "rows": 8192, "vocab": 4096, "n": 20, "dtype": "bf16", "tail": False, "train": True, "temperature": 1.0, "masked": 0.0},
        # an odd vocabulary, so that most rows start off a 16-byte boundary; what the teacher did not list is one outcome
        {"name": "distill_odd", "op": "distill", "rows": 2000, "vocab": 65533, "n": 32, "dtype": "bf16", "tail": True, "train": True, "temperature": 1.5, "masked": 0.1},
        # the losses alone, of a validation set under the largest vocabulary
        {"name": "distill_largest", "op": "distill", "rows": 1024, "vocab": 131072, "n": 64, "dtype": "f32", "tail": True, "train": False, "temperature": 1.0, "masked": 0.0},
        # one song: the sampler's processed scores of four drafted tokens
        {"name": "verify_song", "op": "verify", "rows": 1, "drafts": 4, "vocab": 4096, "dtype": "f32", "mode": "sample", "temperature": 1.0, "masked": 0.5},
        # drafts looked up in what was written before (no draft distribution), sequences of uneven draft lengths
        {"name": "verify_lookup", "op": "verify", "rows": 64, "drafts": 8, "vocab": 4096, "dtype": "bf16", "mode": "lookup", "temperature": 0.9, "masked": 0.0},
        # a batch under a wide vocabulary
        {"name": "verify_wide", "op": "verify", "rows": 64, "drafts": 5, "vocab": 65536, "dtype": "f16", "mode": "sample", "temperature": 0.9, "masked": 0.25},
        # the largest: many sequences, many drafts, the largest vocabulary
        {"name": "verify_largest", "op": "verify", "rows": 128, "drafts": 8, "vocab": 131072, "dtype": "bf16", "mode": "sample", "temperature": 1.0, "masked": 0.0},
    ]


MOST_PRODUCTS = 8192 * 4096 * 16384
MOST_SCORES = 2000 * 65533           # of a distillation step
MOST_VERIFIED = 128 * 17 * 131072    # scores of targets and drafts


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["fp8", "distill", "verify"])
    if op == "fp8":
        rows = _spread(rng, 1, 8192)
        vocab = _spread(rng, 40, min(131072, 134217728 // rows))
        d = _spread(rng, 16, max(16, min(4096, MOST_PRODUCTS // (rows * vocab))))
        if rng.random() < 0.5:  # what models use; the other half is odd
            d, vocab = max(64, d // 64 * 64), max(8, vocab // 8 * 8)
        return {"op": op, "rows": rows, "d": d, "vocab": vocab, "hidden": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "distill":
        rows = _spread(rng, 1, 8192)
        vocab = _spread(rng, 130, min(131072, MOST_SCORES // rows))
        return {"op": op, "rows": rows, "vocab": vocab, "n": rng.choice([1, 5, 20, 32, 50, 128]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "tail": rng.random() < 0.5, "train": rng.random() < 0.7, "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
                "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}
    rows, drafts = _spread(rng, 1, 256), rng.randint(0, 8)
    vocab = _spread(rng, 40, min(131072, MOST_VERIFIED // (rows * (2 * drafts + 1))))
    return {"op": op, "rows": rows, "drafts": drafts, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "mode": rng.choice(["sample", "sample", "lookup", "greedy"]), "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]),
            "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}


def _logits(shape, g, device):
    """A few peaks that hold most of a row's mass over a broad floor, as language models' logits do."""
    vocab = shape[-1]
    x = torch.randn(shape, generator=g, device=device) * 1.5
    peaks = torch.randint(0, vocab, shape[:-1] + (8,), generator=g, device=device)
    return x.scatter_add_(-1, peaks, torch.full(peaks.shape, math.log(vocab) + 1.0, device=device)), peaks


def _near(x, g, noise):
    """Another model's logits of the same positions."""
    return torch.randn(x.shape, generator=g, device=x.device).mul_(noise).add_(x)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    state = {"case": case}
    if case["op"] == "fp8":
        d = case["d"]
        hidden = torch.randn((rows, d), generator=g, device=device)
        hidden[:, :: max(1, d // 6)] *= 6.0  # a few channels are larger, as in trained models
        state["hidden"] = hidden.to(DTYPES[case["hidden"]])
        high, wide = (vocab + BLOCK - 1) // BLOCK, (d + BLOCK - 1) // BLOCK
        weight = torch.zeros((high * BLOCK, wide * BLOCK), device=device)
        weight[:vocab, :d] = torch.randn((vocab, d), generator=g, device=device) * 0.02
        scale = weight.view(high, BLOCK, wide, BLOCK).abs().amax(dim=(1, 3)) / E4M3_MAX
        weight.view(high, BLOCK, wide, BLOCK).div_(scale[:, None, :, None])
        laid = weight[:vocab, : (d + 15) // 16 * 16].clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)  # rows on 16-byte boundaries
        state["weight_q"], state["weight_scale"] = laid[:, :d], scale
        return state
    if case["op"] == "distill":
        n = case["n"]
        base, peaks = _logits((rows, vocab), g, device)
        teacher = _near(base, g, 0.5)
        if case["masked"] > 0:  # ids that the grammar forbids, for both; one stays allowed
            forbidden = torch.rand((rows, vocab), generator=g, device=device) < case["masked"]
            forbidden.scatter_(1, peaks[:, :1], False)
            base.masked_fill_(forbidden, -math.inf)
            teacher.masked_fill_(forbidden, -math.inf)
        teacher = torch.log_softmax(teacher.div_(case["temperature"]), dim=1)
        logprobs, ids = torch.topk(teacher, n, dim=1)
        padded = torch.rand((rows, 1), generator=g, device=device) < 0.1  # positions without a target
        state["teacher_ids"] = ids.masked_fill_(padded | (logprobs == -math.inf), -1)
        state["teacher_logprobs"] = logprobs
        state["logits"] = _near(base, g, 0.5).to(DTYPES[case["dtype"]])
        state["weights"] = torch.rand((rows,), generator=g, device=device) + 0.5
        return state
    drafts, t = case["drafts"], case["temperature"]
    target, peaks = _logits((rows, drafts + 1, vocab), g, device)
    if case["masked"] > 0:
        forbidden = torch.rand(target.shape, generator=g, device=device) < case["masked"]
        forbidden.scatter_(2, peaks[:, :, :1], False)
        target.masked_fill_(forbidden, -math.inf)
    draft = _near(target[:, :drafts], g, 0.7).to(DTYPES[case["dtype"]])
    pick = torch.rand((rows, drafts, vocab), generator=g, device=device).clamp_min_(1e-30).log_().neg_()
    ids = (draft.float() / t).exp_().div_(pick).argmax(dim=2) if drafts else torch.empty((rows, 0), dtype=torch.int64, device=device)
    if case["mode"] == "greedy" and drafts:
        ids = torch.where(torch.rand(ids.shape, generator=g, device=device) < 0.8, target[:, :drafts].argmax(dim=2), ids)
    if case["mode"] == "lookup":  # uneven draft lengths
        length = torch.randint(0, drafts + 1, (rows, 1), generator=g, device=device)
        ids = ids.masked_fill(torch.arange(drafts, device=device) >= length, -1)
    state["draft_ids"] = ids
    state["draft_logits"] = draft if case["mode"] == "sample" else None
    state["target_logits"] = target.to(DTYPES[case["dtype"]])
    state["uniforms"] = torch.rand((rows, drafts + 1), generator=g, device=device)
    return state


def _plain_fp8(hidden, weight_q, weight_scale, dtype):
    rows, d = hidden.shape
    wide = weight_scale.shape[1]
    h = torch.zeros((rows, wide * BLOCK), device=hidden.device)
    h[:, :d] = hidden.float()
    h = h.view(rows, wide, BLOCK)
    scale = h.abs().amax(dim=2) * (1.0 / torch.tensor(E4M3_MAX, device=h.device))
    q = (h / torch.where(scale > 0, scale, 1.0)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).float()
    h = (q * scale[:, :, None]).view(rows, wide * BLOCK)[:, :d]
    each = weight_scale.repeat_interleave(BLOCK, 0)[: weight_q.shape[0]].repeat_interleave(BLOCK, 1)[:, :d]
    return (h @ (weight_q.float() * each).T).to(dtype)


def _plain_distill(state, case):
    ids, lp, t = state["teacher_ids"], state["teacher_logprobs"], case["temperature"]
    x = state["logits"].double() / t  # a loss is a difference of nearly equal logarithms
    z = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(dim=1, keepdim=True)
    given = ids >= 0
    at = ids.clamp_min(0)
    p = torch.where(given, torch.exp(lp.double()), 0.0)
    if not case["tail"]:
        p = p / p.sum(dim=1, keepdim=True).clamp_min(1e-300)
    listed_mass = p.sum(dim=1, keepdim=True)
    of_listed = torch.where(p > 0, p * (torch.log(p) - z.gather(1, at) + torch.log(total)), 0.0)
    loss = of_listed.sum(dim=1)
    outside = torch.ones((x.shape[0], x.shape[1] + 1), dtype=torch.bool, device=x.device)
    outside = outside.scatter_(1, torch.where(given, ids, x.shape[1]), False)[:, :-1]  # the last column takes the missing ids
    rest = torch.where(outside, e, 0.0)
    q_rest = rest.sum(dim=1, keepdim=True) / total
    p_rest = 1.0 - listed_mass if case["tail"] else torch.zeros_like(listed_mass)
    p_rest = torch.where(p_rest < LEAST_REST, 0.0, p_rest)
    loss = loss + torch.where(p_rest > 0, p_rest * (torch.log(p_rest) - torch.log(q_rest)), 0.0)[:, 0]
    none = ~given.any(dim=1)
    loss = torch.where(none, 0.0, loss).float()
    if not case["train"]:
        return loss
    g = torch.where(none, 0.0, state["weights"])[:, None]
    q = (e / total).float()
    even = torch.where(outside, (listed_mass - torch.where(p_rest > 0, p_rest * (1.0 - q_rest) / q_rest, 0.0)).float(), (listed_mass + p_rest).float())
    dx = q * even
    dx.scatter_add_(1, at, -p.float())
    return loss, (dx * g / t).to(state["logits"].dtype)


def _plain_verify(state, case):
    x, ids, u, t = state["target_logits"], state["draft_ids"], state["uniforms"], case["temperature"]
    rows, more, _ = x.shape
    k = more - 1
    z = x.double() / t
    z = z - z.amax(dim=2, keepdim=True)
    logp = z - torch.log(torch.exp(z).sum(dim=2, keepdim=True))
    del z
    p = torch.exp(logp)
    row = torch.arange(rows, device=x.device)
    at = ids.clamp_min(0)[:, :, None]
    if case["mode"] == "greedy":
        best = x.argmax(dim=2)
        accept = (ids == best[:, :k]) & (ids >= 0)
    else:
        if case["mode"] == "sample":
            y = state["draft_logits"].double() / t
            y = torch.exp(y - y.amax(dim=2, keepdim=True))
            q = y / y.sum(dim=2, keepdim=True)
        else:
            q = torch.zeros_like(p[:, :k]).scatter_(2, at, 1.0)
        accept = (u[:, :k].double() * q.gather(2, at)[:, :, 0] < p[:, :k].gather(2, at)[:, :, 0]) & (ids >= 0)
    count = torch.cumprod(accept.long(), dim=1).sum(dim=1)
    if case["mode"] == "greedy":
        last = best[row, count]
    else:
        w = p[row, count]
        if k:
            stop = count.clamp_max(k - 1)
            refused = (count < k) & (ids[row, stop] >= 0)
            w = torch.where(refused[:, None], (w - q[row, stop]).clamp_min(0.0), w)
        run = torch.cumsum(w, dim=1)
        last = (run > (u[:, k].double() * run[:, -1])[:, None]).long().argmax(dim=1)
    tokens = torch.zeros((rows, more), dtype=torch.int64, device=x.device)
    place = torch.arange(k, device=x.device)
    tokens[:, :k] = torch.where(place < count[:, None], ids, 0)
    tokens[row, count] = last
    given = torch.arange(more, device=x.device) <= count[:, None]
    logprobs = torch.where(given, logp.gather(2, tokens[:, :, None])[:, :, 0], 0.0)
    return tokens, count.int(), logprobs.float()


def run(state):
    case = state["case"]
    if case["op"] == "fp8":
        hidden, weight_q, weight_scale, out = state["hidden"], state["weight_q"], state["weight_scale"], DTYPES[case["out"]]
        if own:
            from mapperatorinator_b200.fp8_head import lm_head_logits_fp8

            return lm_head_logits_fp8(hidden, weight_q, weight_scale, out_dtype=out)
        return _plain_fp8(hidden, weight_q, weight_scale, out)
    if case["op"] == "distill":
        if own:
            from mapperatorinator_b200.distillation import distillation_loss, distillation_loss_and_grad

            given = (state["logits"], state["teacher_ids"], state["teacher_logprobs"])
            if not case["train"]:
                return distillation_loss(*given, temperature=case["temperature"], tail=case["tail"])
            return distillation_loss_and_grad(*given, state["weights"], temperature=case["temperature"], tail=case["tail"])
        return _plain_distill(state, case)
    if own:
        from mapperatorinator_b200.speculative import verify_drafts

        greedy = case["mode"] == "greedy"
        r = verify_drafts(state["target_logits"], state["draft_ids"], state["draft_logits"], uniforms=None if greedy else state["uniforms"],
                          temperature=case["temperature"], do_sample=not greedy)
        return r.tokens, r.accepted, r.logprobs
    return _plain_verify(state, case)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "fp8":
        d = case["d"]
        blocks = -(-vocab // BLOCK) * -(-d // BLOCK)
        return {"bytes": rows * d * size[case["hidden"]] + vocab * d + 4 * blocks + rows * vocab * size[case["out"]],
                "flops": 2 * rows * vocab * d}
    if case["op"] == "distill":  # a maximum, a product, an exponential and a sum for each score; two more for its gradient
        one = rows * vocab * size[case["dtype"]]
        train = 1 if case["train"] else 0
        return {"bytes": (1 + train) * one + rows * (12 * case["n"] + 4 + 4 * train), "flops": (4 + 3 * train) * rows * vocab}
    k = case["drafts"]
    scores = rows * (k + 1 + (k if case["mode"] == "sample" else 0)) * vocab
    return {"bytes": scores * size[case["dtype"]] + rows * (8 * k + 4 * (k + 1) + 12 * (k + 1) + 4), "flops": 4 * scores}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "fp8":
        h, wq, ws = state["hidden"].to(torch.float32), state["weight_q"], state["weight_scale"]
        rows, d = h.shape
        logits = torch.zeros((rows, wq.shape[0]), dtype=torch.float64, device=h.device)
        reciprocal = torch.ones((), device=h.device) / E4M3_MAX  # the scale is an fp32 number by definition
        for b in range(ws.shape[1]):
            part = h[:, b * BLOCK : (b + 1) * BLOCK]
            step = torch.linalg.vector_norm(part, math.inf, dim=1, keepdim=True) * reciprocal
            whole = torch.nan_to_num(part / step).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double()
            column = torch.repeat_interleave(ws[:, b].double(), BLOCK)[: wq.shape[0]]
            logits += torch.matmul(whole * step.double(), (wq[:, b * BLOCK : (b + 1) * BLOCK].double() * column[:, None]).t())
        return logits
    if case["op"] == "distill":
        x = state["logits"].double() / case["temperature"]
        x -= torch.logsumexp(x, 1, keepdim=True)  # log q
        ids, lp = state["teacher_ids"], state["teacher_logprobs"].double()
        lp = torch.where(ids < 0, -math.inf, lp)
        if not case["tail"]:
            lp = lp - torch.logsumexp(lp, 1, keepdim=True)
        empty = (ids < 0).all(1)
        lp[empty] = -math.inf
        p = lp.exp()
        # a column behind the vocabulary takes what names no id
        member = torch.zeros((case["rows"], case["vocab"] + 1), dtype=torch.float64, device=x.device)
        member.scatter_add_(1, torch.where(ids < 0, case["vocab"], ids), p)
        inside = torch.zeros_like(member, dtype=torch.bool).scatter_(1, torch.where(ids < 0, case["vocab"], ids), True)[:, :-1]
        member = member[:, :-1]
        cross = torch.where(member > 0, member * x, 0.0).sum(1)
        loss = -torch.special.entr(p).sum(1) - cross
        rest_p = torch.zeros_like(loss)
        rest_logq = torch.logsumexp(x.masked_fill(inside, -math.inf), 1)
        if case["tail"]:
            rest_p = torch.nn.functional.threshold(1.0 - p.sum(1), LEAST_REST * (1.0 - 2.0**-40), 0.0)
            loss = loss + torch.where(rest_p > 0, torch.xlogy(rest_p, rest_p) - rest_p * rest_logq, 0.0)
        loss = loss.masked_fill(empty, 0.0)
        if not case["train"]:
            return loss
        mass = p.sum(1)
        inner = torch.logsumexp(x.masked_fill(~inside, -math.inf), 1).exp()
        slope = x.exp() * torch.where(inside, (mass + rest_p)[:, None], mass[:, None]) - member
        share = torch.where(rest_p > 0, rest_p * inner, 0.0)
        slope -= torch.where(inside | (share == 0)[:, None], 0.0, share[:, None] * (x - torch.where(rest_p > 0, rest_logq, 0.0)[:, None]).exp())
        slope *= (state["weights"].double() / case["temperature"])[:, None]
        return loss, slope.masked_fill(empty[:, None], 0.0)
    k, rows = case["drafts"], case["rows"]
    tokens, counts, scores = [], [], []
    for b in range(rows):  # one sequence after another, as the definition has it
        x = torch.log_softmax(state["target_logits"][b].double() / case["temperature"], 1)
        p, ids, u = x.exp(), state["draft_ids"][b], state["uniforms"][b].double()
        if case["mode"] == "greedy":
            best = state["target_logits"][b].float().argmax(1)
            good = best[:k] == ids
        else:
            q = torch.nn.functional.one_hot(ids.clamp(min=0), case["vocab"]).double()
            if case["mode"] == "sample":
                q = torch.softmax(state["draft_logits"][b].double() / case["temperature"], 1)
            each = torch.arange(k, device=x.device)
            good = (ids >= 0) & (u[:k] * q[each, ids.clamp(min=0)] < p[each, ids.clamp(min=0)])
        n = int(torch.cat([good, good.new_zeros(1)]).long().argmin())
        if case["mode"] == "greedy":
            new = int(best[n])
        else:
            left = p[n]
            if n < k and int(ids[n]) >= 0:
                left = torch.relu(left - q[n])
            sums = left.cumsum(0)
            new = int(torch.searchsorted(sums, (u[k] * sums[-1])[None], right=True))
        line = [int(v) for v in ids[:n]] + [new] + [0] * (k - n)
        given = [float(x[j, line[j]]) if j <= n else 0.0 for j in range(k + 1)]
        tokens.append(line), counts.append(n), scores.append(given)
    device = state["uniforms"].device
    return (torch.tensor(tokens, device=device), torch.tensor(counts, dtype=torch.int32, device=device),
            torch.tensor(scores, dtype=torch.float64, device=device))
