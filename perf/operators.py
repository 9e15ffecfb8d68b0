"""The output head's operators as a user calls them, beside their plain form in elementary torch operations.

  int8   hidden states to logits through an 8-bit output projection: each row of hidden states is quantised
         by its own scale, the weight rows carry theirs (one per vocabulary id)
  score  log probabilities of given tokens, the entropy, the log-sum-exp and the top alternatives of each row
  train  the same without alternatives, and the gradient of the logits
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NO_TOKEN = -100  # a padded position


def listed():
    return [
        # one song: the conditional and unconditional rows of a single step
        {"name": "int8_song", "op": "int8", "rows": 2, "d": 768, "vocab": 4096, "hidden": "bf16", "out": "bf16"},
        # the batched decode's 64 pairs
        {"name": "int8_batch", "op": "int8", "rows": 128, "d": 768, "vocab": 4096, "hidden": "bf16", "out": "bf16"},
        # odd sizes on every axis, half-precision hidden states, fp32 logits
        {"name": "int8_ragged", "op": "int8", "rows": 333, "d": 1001, "vocab": 4099, "hidden": "f16", "out": "f32"},
        # a step of 4096 pairs (the sharded decode on one GPU), or all positions of a few windows
        {"name": "int8_sharded", "op": "int8", "rows": 8192, "d": 768, "vocab": 4096, "hidden": "bf16", "out": "bf16"},
        # the largest vocabulary of the streaming kernel: weights and logits bound
        {"name": "int8_wide", "op": "int8", "rows": 256, "d": 1024, "vocab": 65536, "hidden": "bf16", "out": "bf16"},
        # whole windows through a wide model: bound by the tensor cores
        {"name": "int8_large", "op": "int8", "rows": 8192, "d": 4096, "vocab": 16384, "hidden": "bf16", "out": "bf16"},
        # a served step: emitted tokens under the processed (masked) fp32 scores
        {"name": "score_step", "op": "score", "rows": 64, "vocab": 4096, "dtype": "f32", "top": 5, "masked": 0.5, "temperature": 1.0},
        # all positions of many windows scored
        {"name": "score_windows", "op": "score", "rows": 8192, "vocab": 4096, "dtype": "bf16", "top": 8, "masked": 0.0, "temperature": 1.0},
        # a wide vocabulary, many alternatives, some ids masked by the grammar
        {"name": "score_wide", "op": "score", "rows": 256, "vocab": 65536, "dtype": "f16", "top": 20, "masked": 0.25, "temperature": 0.9},
        # the largest vocabulary in fp32, tokens alone
        {"name": "score_largest", "op": "score", "rows": 1024, "vocab": 131072, "dtype": "f32", "top": 0, "masked": 0.0, "temperature": 1.0},
        # a training step over windows: gradients of log probability, entropy and log-sum-exp together
        {"name": "train_windows", "op": "train", "rows": 8192, "vocab": 4096, "dtype": "bf16", "masked": 0.0, "temperature": 1.0},
        # an odd vocabulary, so that most rows start off a 16-byte boundary
        {"name": "train_odd", "op": "train", "rows": 2000, "vocab": 65533, "dtype": "bf16", "masked": 0.1, "temperature": 0.8},
    ]


MOST_ELEMENTS = 1024 * 131072
MOST_PRODUCTS = 8192 * 4096 * 16384


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["int8", "score", "train"])
    rows = _spread(rng, 1, 8192)
    vocab = _spread(rng, 40, min(131072, MOST_ELEMENTS // rows))
    if op == "int8":
        d = _spread(rng, 16, max(16, min(4096, MOST_PRODUCTS // (rows * vocab))))
        if rng.random() < 0.5:  # what models use; the other half is odd
            d, vocab = max(64, d // 64 * 64), max(8, vocab // 8 * 8)
        return {"op": op, "rows": rows, "d": d, "vocab": vocab, "hidden": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "masked": rng.choice([0.0, 0.0, 0.3, 0.9]), "temperature": rng.choice([1.0, 1.0, 0.7, 1.3])}
    if op == "score":
        case["top"] = rng.choice([0, 1, 5, 8, 20, 32])
    return case


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    state = {"case": case}
    if case["op"] == "int8":
        d = case["d"]
        hidden = torch.randn((rows, d), generator=g, device=device)
        hidden[:, :: max(1, d // 6)] *= 6.0  # a few channels are larger, as in trained models
        state["hidden"] = hidden.to(DTYPES[case["hidden"]])
        weight = torch.randn((vocab, d), generator=g, device=device) * 0.02
        scale = weight.abs().amax(dim=1) / 127.0
        laid = torch.zeros((vocab, (d + 15) // 16 * 16), dtype=torch.int8, device=device)  # rows on 16-byte boundaries
        laid[:, :d] = torch.round(weight / scale[:, None]).to(torch.int8)
        state["weight_q"], state["weight_scale"] = laid[:, :d], scale
        return state
    logits = torch.randn((rows, vocab), generator=g, device=device) * 2.0
    peaks = torch.randint(0, vocab, (rows, 8), generator=g, device=device)
    logits.scatter_add_(1, peaks, torch.full((rows, 8), 6.0, device=device))
    tokens = peaks[:, 0].clone()
    if case["masked"] > 0:  # ids that the grammar forbids; the given token is allowed
        forbidden = torch.rand((rows, vocab), generator=g, device=device) < case["masked"]
        forbidden.scatter_(1, tokens[:, None], False)
        logits.masked_fill_(forbidden, float("-inf"))
    state["logits"] = logits.to(DTYPES[case["dtype"]])
    if case["op"] == "train":
        padded = torch.rand((rows,), generator=g, device=device) < 0.1
        tokens.masked_fill_(padded, NO_TOKEN)
        state["grads"] = (-torch.rand((rows,), generator=g, device=device) - 0.5,          # weights of the log probabilities
                          torch.full((rows,), -0.01, device=device),                         # an entropy bonus
                          torch.rand((rows,), generator=g, device=device) * 1e-2)            # a penalty on the log-sum-exp
        state["logits"].requires_grad_(True)
    state["tokens"] = tokens
    return state


def _plain_int8(hidden, weight_q, weight_scale, dtype):
    h = hidden.float()
    scale = h.abs().amax(dim=1) / 127.0
    q = torch.round(h / torch.where(scale > 0, scale, 1.0)[:, None])
    return ((q @ weight_q.float().T) * scale[:, None] * weight_scale).to(dtype)


def _plain_scores(logits, tokens, temperature):
    """Scaled scores less their maximum, exp of them, its sum, and what `token_logprobs` says of tokens and rows."""
    x = logits.detach().float() / temperature
    top = x.amax(dim=1)
    z = x - torch.where(top.isinf(), 0.0, top)[:, None]
    e = torch.exp(z)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    logp = z - log_total[:, None]
    entropy = -torch.where(e > 0, e * logp, 0.0).sum(dim=1) / total
    given = tokens >= 0
    token_logp = torch.where(given, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    return logp, e / total[:, None], token_logp, entropy, top + log_total


def _plain_top(logits, logp, n):
    value, index = torch.sort(logits.detach().float(), dim=1, descending=True, stable=True)
    value, index = value[:, :n], index[:, :n]
    missing = value == float("-inf")
    return torch.where(missing, -1, index), torch.where(missing, float("-inf"), logp.gather(1, index))


def _plain_gradient(logits, tokens, logp, p, entropy, grads, temperature):
    of_token, of_entropy, of_lse = grads
    of_token = torch.where(tokens >= 0, of_token, 0.0)
    even = (of_lse - of_token - of_entropy * entropy)[:, None]
    dx = p * (even - of_entropy[:, None] * torch.where(p > 0, logp, 0.0))
    dx.scatter_add_(1, tokens.clamp_min(0)[:, None], of_token[:, None])
    return (dx / temperature).to(logits.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "int8":
        hidden, weight_q, weight_scale, out = state["hidden"], state["weight_q"], state["weight_scale"], DTYPES[case["out"]]
        if own:
            from mapperatorinator_b200.int8_head import lm_head_logits_int8

            return lm_head_logits_int8(hidden, weight_q, weight_scale, out_dtype=out)
        return _plain_int8(hidden, weight_q, weight_scale, out)
    logits, tokens, temperature = state["logits"], state["tokens"], case["temperature"]
    if case["op"] == "score":
        if own:
            from mapperatorinator_b200.scoring import token_logprobs

            r = token_logprobs(logits, tokens, top_n=case["top"], temperature=temperature)
            return r.logprobs, r.entropy, r.lse, r.top_ids, r.top_logprobs
        logp, _, token_logp, entropy, lse = _plain_scores(logits, tokens, temperature)
        if not case["top"]:
            return token_logp, entropy, lse, tokens.new_empty((case["rows"], 0)), logp.new_empty((case["rows"], 0))
        return (token_logp, entropy, lse) + _plain_top(logits, logp, case["top"])
    if own:
        from mapperatorinator_b200.scoring import token_logprobs

        r = token_logprobs(logits, tokens, temperature=temperature)
        (grad,) = torch.autograd.grad((r.logprobs, r.entropy, r.lse), logits, state["grads"])
        return r.logprobs.detach(), r.entropy.detach(), r.lse.detach(), grad
    logp, p, token_logp, entropy, lse = _plain_scores(logits, tokens, temperature)
    return token_logp, entropy, lse, _plain_gradient(logits, tokens, logp, p, entropy, state["grads"], temperature)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "int8":
        d = case["d"]
        return {"bytes": rows * d * size[case["hidden"]] + vocab * (d + 4) + rows * vocab * size[case["out"]],
                "flops": 2 * rows * vocab * d}
    one = rows * vocab * size[case["dtype"]]
    if case["op"] == "score":  # a maximum, an exponential, two sums and a product for each score
        return {"bytes": one + rows * (8 + 12 + 12 * case["top"]), "flops": 6 * rows * vocab}
    return {"bytes": 2 * one + rows * (8 + 12 + 12), "flops": 12 * rows * vocab}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "int8":
        h = state["hidden"].to(torch.float32)
        step = torch.max(torch.abs(h), 1).values / 127.0  # the scale is an fp32 number by definition
        whole = torch.nan_to_num(h.double() / step.double().unsqueeze(1)).round()
        dot = torch.matmul(whole, state["weight_q"].double().t())
        return dot.mul_(step.double().unsqueeze(1)).mul_(state["weight_scale"].double().unsqueeze(0))
    x = state["logits"].detach().double().div_(case["temperature"])
    lse = torch.logsumexp(x, 1)
    x.sub_(lse.unsqueeze(1))  # log p
    at = state["tokens"]
    kept = (at >= 0).double()
    of_given = x[torch.arange(case["rows"], device=x.device), at.clamp(min=0)]
    spread = torch.special.entr(x.exp()).sum(1)
    given = torch.where(at >= 0, of_given, torch.zeros_like(of_given))
    if case["op"] == "score":
        n = case["top"]
        room = torch.full((case["rows"], max(0, n - case["vocab"])), -math.inf, device=x.device, dtype=x.dtype)
        best = torch.cat([torch.topk(x, min(n, case["vocab"]), 1).values, room], 1)
        return given, spread, lse, None, best
    w, b, z = (v.double() for v in state["grads"])
    p = x.exp()
    # d H / d x_v = -p_v (log p_v + H), d lse / d x_v = p_v, d log p_t / d x_v = [v = t] - p_v
    slope = torch.special.entr(p).sub_(p * spread.unsqueeze(1)).mul_(b.unsqueeze(1)).add_(p * (z - w * kept).unsqueeze(1))
    slope[torch.arange(case["rows"], device=x.device), at.clamp(min=0)] += w * kept
    return given, spread, lse, slope.div_(case["temperature"])
