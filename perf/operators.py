"""Measured cases of the scored router, the 8-bit integer products and the token log probabilities.

``run`` computes an operator either in its plain form (elementary torch operations) or, where ``own`` is true, through
the framework's entry points:

* ``route``: scores of T rows of router logits (softmax or sigmoid), a balance bias that moves the choice but not the
  weights, groups of experts, the top k and their renormalised weights (``yanah_b200.routing.route_scored``);
* ``linear``: rows quantised to 8-bit integers with one scale per row, times a matrix of 8-bit integers with one scale
  per output channel (``yanah_b200.int8.int8_linear``);
* ``experts``: the routed experts of an MoE layer in that form, gate / up, SwiGLU, down, the weighted sum over a row's
  experts and the residual (``yanah_b200.int8.int8_experts``);
* ``logprobs``: log probability and rank of a given token per row, the row's entropy and its likeliest alternatives
  (``yanah_b200.logprobs.token_logprobs``).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}

#: (experts, top k, hidden, intermediate) of the framework's two synthetic stacks, of its test configuration and of
#: two odd ones.
EXPERT_SHAPES = ((512, 10, 2048, 512), (64, 4, 2048, 1536), (64, 4, 1024, 256), (24, 3, 1000, 360), (40, 6, 712, 333))


def listed():
    return [
        # One decode step of the 512-expert stack: the smallest call, all latency.
        {"op": "route", "name": "route_1x512_softmax", "rows": 1, "experts": 512, "k": 10, "score": "softmax",
         "bias": False, "groups": 1, "kept": 1, "masked": 0.0, "dtype": "fp32"},
        # A ragged batch of prompt rows (37 + 300 + 5) of the 64-expert stack, with a balance bias.
        {"op": "route", "name": "route_342x64_sigmoid_bias", "rows": 342, "experts": 64, "k": 4, "score": "sigmoid",
         "bias": True, "groups": 1, "kept": 1, "masked": 0.0, "dtype": "fp32"},
        # A large prompt pass whose experts live in 8 groups (nodes), of which a row may use 4.
        {"op": "route", "name": "route_16384x256_groups", "rows": 16384, "experts": 256, "k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "masked": 0.0, "dtype": "bf16"},
        # The LM head of one decoded token.
        {"op": "linear", "name": "linear_1x2048x65536", "rows": 1, "k": 2048, "n": 65536, "dtype": "bf16",
         "out": "fp32"},
        # The LM head of a verify pass (1 + 4 draft rows) with a large vocabulary.
        {"op": "linear", "name": "linear_5x2048x151936", "rows": 5, "k": 2048, "n": 151936, "dtype": "bf16",
         "out": "fp32"},
        # A projection of a large prompt pass: bound by the tensor cores.
        {"op": "linear", "name": "linear_4096x2048x16384", "rows": 4096, "k": 2048, "n": 16384, "dtype": "bf16",
         "out": "bf16"},
        # The routed experts of one decoded token (512-expert stack).
        {"op": "experts", "name": "experts_1x512", "rows": 1, "shape": 0, "absent": 0.0, "dtype": "bf16"},
        # A decode batch of 250 sequences: nearly every expert is read, most of them for a few rows.
        {"op": "experts", "name": "experts_250x512", "rows": 250, "shape": 0, "absent": 0.0, "dtype": "bf16"},
        # A prompt pass of the 64-expert stack: hundreds of rows per expert, ragged.
        {"op": "experts", "name": "experts_4096x64", "rows": 4096, "shape": 1, "absent": 0.0, "dtype": "bf16"},
        # The answer of one decoded token with 20 alternatives.
        {"op": "logprobs", "name": "logprobs_1x151936", "rows": 1, "vocab": 151936, "top": 20, "masked": 0.0,
         "pad": 0, "dtype": "fp32"},
        # The verify rows' answers over an odd vocabulary in padded rows, a part of it barred from sampling.
        {"op": "logprobs", "name": "logprobs_5x100003", "rows": 5, "vocab": 100003, "top": 5, "masked": 0.1,
         "pad": 61, "dtype": "fp32"},
        # Scoring a prompt: every position's token, as evaluation and logprob requests do.
        {"op": "logprobs", "name": "logprobs_4096x65536", "rows": 4096, "vocab": 65536, "top": 8, "masked": 0.0,
         "pad": 0, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("route", "linear", "experts", "logprobs"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        per = _spread(rng, 2 if groups > 1 else 8, 512 // groups)
        experts = groups * per
        kept = rng.randint(1, groups)
        return {"op": op, "rows": _spread(rng, 1, min(16384, 16384 * 256 // experts)), "experts": experts,
                "k": rng.randint(1, min(16, kept * per)), "score": rng.choice(("softmax", "sigmoid")),
                "bias": rng.random() < 0.6, "groups": groups, "kept": kept,
                "masked": rng.choice((0.0, 0.0, 0.2, 0.9)), "dtype": rng.choice(("fp32", "bf16", "fp16"))}
    if op == "linear":
        k = _spread(rng, 48, 4096)
        n = _spread(rng, 64, min(151936, 2048 * 151936 // k))
        return {"op": op, "rows": _spread(rng, 1, min(4096, 4096 * 2048 * 16384 // (k * n))), "k": k, "n": n,
                "dtype": rng.choice(("bf16", "fp16", "fp32")), "out": rng.choice(("bf16", "fp32", "fp16"))}
    if op == "experts":
        shape = rng.randrange(len(EXPERT_SHAPES))
        return {"op": op, "rows": _spread(rng, 1, min(4096, 10000 // EXPERT_SHAPES[shape][1])), "shape": shape,
                "absent": rng.choice((0.0, 0.0, 0.3)), "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    vocab = _spread(rng, 257, 151936)
    return {"op": op, "rows": _spread(rng, 1, min(4096, 4096 * 65536 // (2 * vocab))), "vocab": vocab,
            "top": rng.choice((0, 1, 5, 8, 20)), "masked": rng.choice((0.0, 0.1, 0.95)),
            "pad": rng.choice((0, 0, 1, 61)), "dtype": rng.choice(("fp32", "bf16", "fp16"))}


def _codes(g, lead, cols):
    """Codes of a trained matrix's rows (near normal, the largest near 127), rows starting at multiples of 16 bytes."""
    padded = torch.empty(*lead, (cols + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    codes = padded[..., :cols]
    codes.copy_(torch.randn(*lead, cols, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127))
    return codes


def _scales(g, lead, cols):
    """Channel scales that give the dequantised rows a norm near one."""
    return (1 + 0.2 * torch.rand(*lead, generator=g, device="cuda")) / (32 * math.sqrt(cols))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    state = {"case": case}
    op, rows = case["op"], case["rows"]
    if op == "route":
        e = case["experts"]
        z = 1.3 * normal(rows, e)
        available = None
        if case["masked"]:
            # one per cent of the logits barred row by row, and whole experts that are away
            z = z.masked_fill(torch.rand(rows, e, generator=g, device="cuda") < 0.01, -math.inf)
            available = torch.rand(e, generator=g, device="cuda") >= case["masked"]
        state["logits"] = z.to(DTYPES[case["dtype"]])
        state["bias"] = 0.1 * normal(e) if case["bias"] else None
        state["available"] = available
    elif op == "linear":
        state["x"] = (normal(rows, case["k"]) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))).to(
            DTYPES[case["dtype"]])
        state["codes"], state["scales"] = _codes(g, (case["n"],), case["k"]), _scales(g, (case["n"],), case["k"])
    elif op == "experts":
        e, k, h, i = EXPERT_SHAPES[case["shape"]]
        state["x"] = normal(rows, h).to(DTYPES[case["dtype"]])
        state["residual"] = normal(rows, h).to(DTYPES[case["dtype"]])
        # routing as the synthetic stacks have it: popularity near Zipf, a row's experts distinct
        pop = -1.1 * torch.log(1.0 + torch.randperm(e, generator=g, device="cuda").float())
        z = 1.3 * normal(rows, e) + pop
        top, ids = torch.topk(z, k, dim=1)
        state["weights"] = torch.softmax(top, 1)
        ids = ids.int()
        if case["absent"]:
            ids = ids.masked_fill(torch.rand(rows, k, generator=g, device="cuda") < case["absent"], -1)
        state["ids"] = ids
        for name, lead, cols in (("gate", (e, i), h), ("up", (e, i), h), ("down", (e, h), i)):
            state[name], state[name + "_scales"] = _codes(g, lead, cols), _scales(g, lead, cols)
    else:
        v = case["vocab"]
        z = torch.empty(rows, v + case["pad"], dtype=DTYPES[case["dtype"]], device="cuda")
        z.copy_(2.5 * normal(rows, v + case["pad"]))
        logits = z[:, :v]
        # a few likely tokens per row stand out, as a language model's do
        likely = torch.randint(0, v // 12, (rows, 12), generator=g, device="cuda")
        likely += v // 12 * torch.arange(12, device="cuda")
        logits.scatter_(1, likely, (4 * normal(rows, 12) + 11).to(z.dtype))
        if case["masked"]:
            logits.masked_fill_(torch.rand(v, generator=g, device="cuda") < case["masked"], -math.inf)
        tokens = likely[:, 0].clone()
        tokens[1::3] = torch.randint(0, v, (rows,), generator=g, device="cuda")[1::3]
        state["logits"], state["tokens"] = logits, tokens.int()
    return state


# ------------------------------------------------------------------------------------------------------ plain forms
def _route_plain(s):
    """Scores and choices in 64 bits (the order of near-equal choices is a border), one rounding of the weights."""
    c = s["case"]
    z = s["logits"].double()
    rows, e = z.shape
    ok = ~torch.isnan(z) & (z != -math.inf)
    if s["available"] is not None:
        ok = ok & s["available"]
    z = z.masked_fill(~ok, -math.inf)
    if c["score"] == "softmax":
        p = torch.exp(z - z.amax(1, keepdim=True).clamp(min=-1e300))
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        p = 1 / (1 + torch.exp(-z))
    pick = z if s["bias"] is None and c["groups"] == 1 else p if s["bias"] is None else p + s["bias"].double()
    pick = pick.masked_fill(~ok, -math.inf)
    if c["groups"] > 1:
        best = torch.sort(pick.view(rows, c["groups"], -1), dim=2, descending=True).values[:, :, :2]
        score = best.masked_fill(best == -math.inf, 0).sum(2).masked_fill(best[:, :, 0] == -math.inf, -math.inf)
        keep = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :c["kept"]]
        kept = torch.zeros_like(score, dtype=torch.bool).scatter_(1, keep, True)
        pick = pick.masked_fill(~kept.repeat_interleave(e // c["groups"], 1), -math.inf)
    value, ids = torch.sort(pick, dim=1, descending=True, stable=True)
    value, ids = value[:, :c["k"]], ids[:, :c["k"]]
    some = value != -math.inf
    w = p.gather(1, ids).masked_fill(~some, 0)
    w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return {"ids": ids.masked_fill(~some, -1).int(), "weights": (w * 2.5).float()}


def _quantise_plain(x):
    """Row codes (whole numbers in fp32) and scales: 127 x / max|x|, ties to even. The quotient in 64 bits: in 32 a
    value next to the border between two codes would fall to the other side of it."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(127 * x.double() / torch.where(top > 0, top, 1).double()).float(), top / 127


def _linear_plain(s):
    q, scale = _quantise_plain(s["x"])
    return ((q @ s["codes"].float().t()) * scale * s["scales"]).to(DTYPES[s["case"]["out"]])


BLOCK = 64  # rows of one expert that the plain form multiplies at once


def _experts_plain(s):
    """Pairs (row, expert) sorted by expert and padded to blocks of one expert each; batched products over the
    blocks. With fewer pairs than experts each pair is a block of one row."""
    x, ids, w = s["x"].float(), s["ids"].long(), s["weights"]
    rows, k = ids.shape
    e, h = s["gate"].shape[0], x.shape[1]
    block = 1 if rows * k < e else BLOCK
    flat = ids.flatten()
    count = torch.zeros(e + 1, dtype=torch.long, device=x.device).scatter_add_(
        0, torch.where(flat < 0, e, flat), torch.ones_like(flat))
    order = torch.sort(torch.where(flat < 0, e, flat), stable=True).indices
    expert = torch.where(flat < 0, e, flat)[order]
    blocks = (count[:e] + block - 1) // block
    first = torch.cumsum(blocks, 0) - blocks
    start = torch.cumsum(count, 0) - count
    n_blocks = rows * k // block + (e if block > 1 else 0)
    place = torch.arange(rows * k, device=x.device) - start[expert]
    place = torch.where(expert < e, torch.cat((first, first[:1]))[expert] * block + place, n_blocks * block)
    of_block = torch.searchsorted(torch.cumsum(blocks, 0), torch.arange(n_blocks, device=x.device), right=True)
    of_block = of_block.clamp(max=e - 1)
    q, scale = _quantise_plain(x)
    pq = torch.zeros(n_blocks * block + 1, h, device=x.device).index_copy_(0, place, q[order // k])
    ps = torch.zeros(n_blocks * block + 1, 1, device=x.device).index_copy_(0, place, scale[order // k])
    pq, ps = pq[:-1].view(n_blocks, block, h), ps[:-1].view(n_blocks, block, 1)

    def times(a, scale, name):
        y = torch.bmm(a, s[name][of_block].float().transpose(1, 2))
        return y * scale * s[name + "_scales"][of_block].unsqueeze(1)

    gate, up = times(pq, ps, "gate"), times(pq, ps, "up")
    act = gate / (1 + torch.exp(-gate)) * up
    y = times(*_quantise_plain(act), "down").view(-1, h)
    y = torch.cat((y, y.new_zeros(1, h)))
    back = torch.empty_like(place).scatter_(0, order, place)
    y = y[back].view(rows, k, h) * torch.where(ids >= 0, w, 0).unsqueeze(2)
    return (s["residual"].float() + y.sum(1)).to(s["x"].dtype)


def _logprobs_plain(s):
    n = s["case"]["top"]
    z = s["logits"].float()
    rows, v = z.shape
    top, first = z.max(1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    # the sum without its largest term, which is one: the logarithm stays exact where that term is nearly all
    rest = e.scatter(1, first, 0).sum(1, keepdim=True)
    total, log_total = 1 + rest, torch.log1p(rest)
    tok = s["tokens"].long().unsqueeze(1)
    at = z.gather(1, tok)
    place = torch.arange(v, device=z.device)
    rank = ((z > at) | ((z == at) & (place < tok))).sum(1).int()
    entropy = log_total - (e * d.masked_fill(e == 0, 0)).sum(1, keepdim=True) / total
    out = {"logprob": (at - top - log_total).squeeze(1), "entropy": entropy.squeeze(1), "rank": rank}
    if n:
        # keys of 64 bits: the value's order above, the lower token first among equal values
        bits = (z + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (v - 1 - place)
        best = torch.topk(key, n, dim=1).indices
        value = z.gather(1, best)
        out["top_ids"] = best.masked_fill(value == -math.inf, -1).int()
        out["top_logprobs"] = value - top - log_total
    return out


def run(state):
    c = state["case"]
    if own:
        if c["op"] == "route":
            from yanah_b200.routing import RouteRule, route_scored
            rule = RouteRule(top_k=c["k"], score=c["score"], n_groups=c["groups"], top_groups=c["kept"], scale=2.5)
            ids, weights = route_scored(state["logits"], rule, bias=state["bias"], available=state["available"])
            return {"ids": ids, "weights": weights}
        if c["op"] == "linear":
            from yanah_b200.int8 import Int8Matrix, int8_linear
            return int8_linear(state["x"], Int8Matrix(state["codes"], state["scales"]), out_dtype=DTYPES[c["out"]])
        if c["op"] == "experts":
            from yanah_b200.int8 import Int8Matrix, int8_experts
            return int8_experts(state["x"], state["ids"], state["weights"],
                                Int8Matrix(state["gate"], state["gate_scales"]),
                                Int8Matrix(state["up"], state["up_scales"]),
                                Int8Matrix(state["down"], state["down_scales"]), residual=state["residual"])
        from yanah_b200.logprobs import token_logprobs
        r = token_logprobs(state["logits"], state["tokens"], n_top=c["top"])
        out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
        if c["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if c["op"] == "route":
        return _route_plain(state)
    if c["op"] == "linear":
        return _linear_plain(state)
    if c["op"] == "experts":
        return _experts_plain(state)
    return _logprobs_plain(state)


def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        e = case["experts"]
        return {"bytes": rows * e * SIZES[case["dtype"]] + 4 * e * case["bias"] + 8 * rows * case["k"],
                "flops": 4 * rows * e}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": rows * k * SIZES[case["dtype"]] + n * k + 4 * n + rows * n * SIZES[case["out"]],
                "flops": 2 * rows * k * n}
    if case["op"] == "experts":
        e, k, h, i = EXPERT_SHAPES[case["shape"]]
        pairs = rows * k * (1 - case["absent"])
        # the experts that a batch reads: all but those that no pair chose, were the choice even
        used = e * (1 - (1 - 1 / e) ** pairs)
        return {"bytes": used * (3 * h * i + 4 * (2 * i + h)) + rows * (3 * h * 2 + 8 * k), "flops": 6 * pairs * h * i}
    v = case["vocab"]
    return {"bytes": rows * v * SIZES[case["dtype"]] + rows * (16 + 8 * case["top"]), "flops": 5 * rows * v}


# ---------------------------------------------------------------------------------------------- the same in 64 bits
def _route_exact(s):
    c = s["case"]
    z = s["logits"].cpu().double().numpy()
    import numpy as np
    rows, e = z.shape
    away = np.isnan(z) | np.isneginf(z)
    if s["available"] is not None:
        away |= ~s["available"].cpu().numpy()[None, :]
    z = np.where(away, -np.inf, z)
    with np.errstate(invalid="ignore", over="ignore"):
        if c["score"] == "softmax":
            p = np.exp(z - np.maximum(z.max(1, keepdims=True), -1e300))
            p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
        else:
            p = 1 / (1 + np.exp(-z))
    order = p + (0 if s["bias"] is None else s["bias"].cpu().double().numpy()[None, :])
    order = np.where(away, -np.inf, order)
    g, n = c["groups"], e // c["groups"]
    if g > 1:
        two = -np.sort(-order.reshape(rows, g, n), axis=2)[:, :, :2]
        sums = np.where(np.isneginf(two), 0, two).sum(2)
        sums[np.isneginf(two[:, :, 0])] = -np.inf
        chosen = np.argsort(-sums, axis=1, kind="stable")[:, :c["kept"]]
        shut = np.ones((rows, g), bool)
        np.put_along_axis(shut, chosen, False, 1)
        order = np.where(np.repeat(shut, n, 1), -np.inf, order)
    elif s["bias"] is None:
        order = z
    ids = np.argsort(-order, axis=1, kind="stable")[:, :c["k"]]
    gone = np.isneginf(np.take_along_axis(order, ids, 1))
    w = np.where(gone, 0, np.take_along_axis(p, ids, 1))
    w = 2.5 * w / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return {"ids": np.where(gone, -1, ids).astype(np.int32), "weights": w}


def _rows64(x):
    """Codes and scales of rows, from the definition: the nearest whole number to 127 x / max|x|."""
    x = x.double()
    peak = x.abs().max(dim=1, keepdim=True).values
    ratio = x * 127 / peak.clamp(min=torch.finfo(torch.float64).tiny)
    return torch.round(ratio), peak / 127


def _linear_exact(s):
    q, scale = _rows64(s["x"])
    parts = [q @ c.double().T * scale * f.double() for c, f in zip(s["codes"].split(16384), s["scales"].split(16384))]
    return torch.cat(parts, 1)


def _experts_exact(s):
    q, scale = _rows64(s["x"])
    out = s["residual"].double()
    for e in range(s["gate"].shape[0]):
        t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not len(t):
            continue
        gate = q[t] @ s["gate"][e].double().T * scale[t] * s["gate_scales"][e].double()
        up = q[t] @ s["up"][e].double().T * scale[t] * s["up_scales"][e].double()
        a, a_scale = _rows64(gate * torch.sigmoid(gate) * up)
        y = a @ s["down"][e].double().T * a_scale * s["down_scales"][e].double()
        out.index_add_(0, t, y * s["weights"][t, j].double().unsqueeze(1))
    return out


def _logprobs_exact(s):
    n, parts = s["case"]["top"], []
    for z, tok in zip(s["logits"].split(256), s["tokens"].split(256)):
        lp = torch.log_softmax(z.double(), 1)
        p = torch.exp(lp)
        at = lp.gather(1, tok.long().unsqueeze(1)).squeeze(1)
        entropy = -(p * torch.where(p > 0, lp, 0)).sum(1)
        best = torch.sort(lp, dim=1, descending=True).values[:, :n]
        parts.append((at, entropy, best))
    at, entropy, best = (torch.cat(v) for v in zip(*parts))
    out = {"logprob": at, "entropy": entropy, "rank": None}
    if n:
        out["top_ids"], out["top_logprobs"] = None, best
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _route_exact, "linear": _linear_exact, "experts": _experts_exact,
            "logprobs": _logprobs_exact}[case["op"]](state)
