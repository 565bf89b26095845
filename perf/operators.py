"""What the operators of a mixture-of-experts language model cost: the router
(``route_experts``), the experts' gated products (``expert_mlp``) and the reading of
the answer (``token_logprobs``), each as one call, with its plain form in elementary
torch operations and its definition in 64 bits.

``own`` chooses what ``run`` calls: the framework's entry points, or the plain form.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One token's router logits while an answer is written: only latency counts.
        dict(name="route_token", op="route", tokens=1, experts=64, top_k=8, score="softmax", bias=False, groups=1,
             top_groups=1, group_top=1, renormalize=True, scale=1.0, dtype="f32", masked=0.0),
        # A serving batch's tokens in 16-bit logits, groups limited by their best expert,
        # some experts switched off for some tokens; sizes that fill no warp.
        dict(name="route_batch", op="route", tokens=1001, experts=160, top_k=6, score="softmax", bias=False, groups=8,
             top_groups=3, group_top=1, renormalize=False, scale=16.0, dtype="bf16", masked=0.05),
        # A long prompt: sigmoid scores, a balancing bias, groups ranked by their two best.
        dict(name="route_prompt", op="route", tokens=16384, experts=256, top_k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, group_top=2, renormalize=True, scale=2.5, dtype="f32", masked=0.0),
        # One token through its eight experts: the weights' bytes and latency.
        dict(name="mlp_token", op="mlp", tokens=1, hidden=2048, inner=1024, experts=64, top_k=8, dtype="bf16",
             dropped=0.0),
        # A decode batch: nearly every expert is read for a handful of rows.
        dict(name="mlp_batch", op="mlp", tokens=48, hidden=2048, inner=1024, experts=64, top_k=8, dtype="bf16",
             dropped=0.0),
        # Ragged everything: few experts, sizes off the tiles, pairs that other ranks take.
        dict(name="mlp_ragged", op="mlp", tokens=777, hidden=1032, inner=688, experts=10, top_k=2, dtype="f16",
             dropped=0.1),
        # Long prompts together: bound by the products.
        dict(name="mlp_prompt", op="mlp", tokens=8192, hidden=2048, inner=1024, experts=64, top_k=8, dtype="bf16",
             dropped=0.0),
        # The sampled token's log probability with alternatives, one sequence.
        dict(name="logprobs_token", op="logprobs", rows=1, vocabulary=128000, top=20, scale=1.0, dtype="bf16",
             masked=0.0, pad=0),
        # A decode batch in 32 bits, an odd vocabulary in padded rows.
        dict(name="logprobs_batch", op="logprobs", rows=96, vocabulary=50001, top=5, scale=1.25, dtype="f32",
             masked=0.0, pad=47),
        # Answers under a grammar: most of the vocabulary masked, log probabilities of the given tokens only.
        dict(name="logprobs_masked", op="logprobs", rows=1500, vocabulary=32003, top=0, scale=1.0, dtype="f16",
             masked=0.6, pad=13),
        # Scoring whole prompts.
        dict(name="logprobs_prompt", op="logprobs", rows=4096, vocabulary=128000, top=20, scale=1.0, dtype="bf16",
             masked=0.0, pad=0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "mlp", "logprobs"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _spread(rng, 8 // groups + 1, 512 // groups)
        top_groups = rng.randint((groups + 1) // 2, groups)
        score = rng.choice(["softmax", "sigmoid"])
        return dict(op=op, tokens=_spread(rng, 1, 16384 * 256 // max(experts, 256)), experts=experts,
                    top_k=rng.randint(1, min(10, top_groups * (experts // groups))), score=score,
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_top=rng.choice([1, 2]),
                    renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                    dtype=rng.choice(["f32", "bf16", "f16"]), masked=rng.choice([0.0, 0.0, 0.1]))
    if op == "mlp":
        hidden, inner = 8 * _spread(rng, 16, 256), 16 * _spread(rng, 4, 64)
        experts = _spread(rng, 4, 64)
        return dict(op=op, tokens=_spread(rng, 1, 8192), hidden=hidden, inner=inner, experts=experts,
                    top_k=rng.randint(1, min(8, experts)), dtype=rng.choice(["bf16", "f16"]),
                    dropped=rng.choice([0.0, 0.0, 0.25]))
    vocabulary = _spread(rng, 1000, 128000)
    return dict(op=op, rows=_spread(rng, 1, 4096), vocabulary=vocabulary, top=rng.choice([0, 1, 5, 20]),
                scale=rng.choice([1.0, 1.25]), dtype=rng.choice(["bf16", "f16"] if vocabulary > 60000 else
                                                               ["bf16", "f16", "f32"]),
                masked=rng.choice([0.0, 0.0, 0.5]), pad=rng.choice([0, 0, 8, 21]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        logits = (normal(t, e) * 1.5 + normal(e) * 0.5).to(dtype)
        if case["masked"]:
            logits.masked_fill_(torch.rand(t, e, generator=g, device="cuda") < case["masked"], -math.inf)
        state["logits"] = logits
        # a balancing bias moves in steps of one thousandth
        state["bias"] = torch.round(normal(e) * 50) / 1000 if case["bias"] else None
    elif case["op"] == "mlp":
        t, e, k, d, f = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inner"))
        scores = normal(t, e) + normal(e) * 0.4  # some experts are liked more than others
        top = torch.topk(scores, k, dim=1)
        ids = top.indices.to(torch.int32)
        if case["dropped"]:
            ids.masked_fill_(torch.rand(t, k, generator=g, device="cuda") < case["dropped"], -1)
        state["ids"] = ids
        state["weights"] = torch.softmax(top.values, dim=1)
        state["x"] = normal(t, d).to(dtype)
        gate_up = torch.empty(e, 2 * f, d, dtype=dtype, device="cuda").normal_(0, d ** -0.5, generator=g)
        state["gate_up"] = gate_up
        state["down"] = torch.empty(e, d, f, dtype=dtype, device="cuda").normal_(0, f ** -0.5, generator=g)
        # the most rows that one expert has: the capacity that a padded plain program plans for
        state["capacity"] = max(1, int(torch.bincount(ids[ids >= 0].long(), minlength=e).max()))
    else:
        n, v = case["rows"], case["vocabulary"]
        rows = torch.empty(n, v + case["pad"], dtype=dtype, device="cuda")
        logits = rows[:, :v]
        torch.mul(normal(n, v), 2.5, out=logits) if dtype == torch.float32 else logits.copy_(normal(n, v) * 2.5)
        if case["masked"]:
            logits.masked_fill_(torch.rand(n, v, generator=g, device="cuda") < case["masked"], -math.inf)
        state["logits"] = logits
        # the given tokens: likely ones, as a model's own answers are
        pick = torch.randint(v, (n, 64), generator=g, device="cuda")
        state["tokens"] = pick.gather(1, logits.gather(1, pick).float().argmax(1, keepdim=True)).squeeze(1)
    return state


def run(state):
    if state["op"] == "route":
        args = (state["logits"], state["top_k"])
        options = dict(score=state["score"], bias=state["bias"], groups=state["groups"],
                       top_groups=state["top_groups"], group_top=state["group_top"],
                       renormalize=state["renormalize"], scale=state["scale"])
        if own:
            import thintnpu_b200
            return thintnpu_b200.route_experts(*args, **options)
        return _route(*args, **options)
    if state["op"] == "mlp":
        if own:
            import thintnpu_b200
            return thintnpu_b200.expert_mlp(state["x"], state["ids"], state["weights"], state["gate_up"],
                                            state["down"])
        return _mlp(state["x"], state["ids"], state["weights"], state["gate_up"], state["down"], state["capacity"])
    if own:
        import thintnpu_b200
        return thintnpu_b200.token_logprobs(state["logits"], state["tokens"], top=state["top"], scale=state["scale"])
    return _logprobs(state["logits"], state["tokens"], state["top"], state["scale"])


def _first(order, count):
    """The leading columns of a stable descending order."""
    return torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :count]


def _route(logits, top_k, *, score, bias, groups, top_groups, group_top, renormalize, scale):
    t, e = logits.shape
    x = logits.double()  # neighbours at the border of the choice differ by less than 32 bits hold
    open_ = logits != -math.inf
    if score == "softmax":
        raised = torch.exp(x - x.amax(1, keepdim=True))
        s = raised / raised.sum(1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-x))
    rank = s if bias is None else s + bias.double()
    rank = torch.where(open_, rank, -math.inf)
    if groups > 1:
        inside = rank.view(t, groups, e // groups)
        best = torch.sort(inside, dim=2, descending=True).values[..., :group_top]
        total = torch.where(best == -math.inf, 0, best).sum(2)
        total = torch.where(best[..., 0] == -math.inf, -math.inf, total)
        kept = torch.zeros(t, groups, dtype=torch.bool, device=x.device)
        kept.scatter_(1, _first(total, top_groups), True)
        rank = torch.where(kept[..., None], inside, -math.inf).view(t, e)
    ids = _first(rank, top_k)
    taken = rank.gather(1, ids) != -math.inf
    w = torch.where(taken, s.gather(1, ids), 0)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0)
    return (w * scale).float(), torch.where(taken, ids, -1).to(torch.int32)


def _mlp(x, ids, weights, gate_up, down, capacity):
    t, k = ids.shape
    e, d, f = down.shape
    pair = ids.reshape(-1).long()
    kept = pair >= 0
    rows = x.float().repeat_interleave(k, 0)
    if t * k <= e:  # fewer pairs than experts: each pair with its own copy of its expert's weights
        at = pair.clamp(min=0)
        both = torch.bmm(gate_up[at].float(), rows[:, :, None])[..., 0]
        y = torch.bmm(down[at].float(), (_silu(both[:, :f]) * both[:, f:])[:, :, None])[..., 0]
    else:  # rows in one padded block for each expert
        slot = torch.where(kept, pair, e)
        order = torch.argsort(slot, stable=True)
        count = torch.zeros(e + 1, dtype=torch.long, device=x.device).scatter_add_(0, slot, torch.ones_like(slot))
        start = torch.cumsum(count, 0) - count
        place = torch.empty_like(order)
        place[order] = torch.arange(t * k, device=x.device) - start[slot[order]]
        place = torch.where(kept, place, 0)
        blocks = torch.zeros(e + 1, capacity, d, dtype=torch.float32, device=x.device)
        blocks[slot, place] = rows
        both = torch.bmm(blocks[:e], gate_up.float().transpose(1, 2))
        y = torch.bmm(_silu(both[..., :f]) * both[..., f:], down.float().transpose(1, 2))
        y = y[torch.where(kept, pair, 0), place]
    y = torch.where(kept[:, None], y * weights.reshape(-1, 1), 0)
    return y.view(t, k, d).sum(1).to(x.dtype)


def _silu(v):
    return v / (1 + torch.exp(-v))


def _logprobs(logits, tokens, top, scale):
    n, v = logits.shape
    x = logits.float() * scale
    shifted = x - x.amax(1, keepdim=True)
    raised = torch.exp(shifted)
    total = raised.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - torch.where(raised > 0, raised * shifted, 0).sum(1) / total[:, 0]
    given = (shifted.gather(1, tokens[:, None]) - log_total)[:, 0]
    # one whole-number key for value and place: larger values first, then lower places
    bits = logits.float().view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32) + (v - 1 - torch.arange(v, device=x.device))
    place = v - 1 - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
    values = shifted.gather(1, place) - log_total
    return given, entropy, values, torch.where(values == -math.inf, -1, place).to(torch.int32)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        return {"bytes": t * e * size + t * case["top_k"] * 8 + (4 * e if case["bias"] else 0), "flops": 4 * t * e}
    if case["op"] == "mlp":
        t, e, k, d, f = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inner"))
        kept = t * k * (1 - case["dropped"])
        read = e * (1 - (1 - k * (1 - case["dropped"]) / e) ** t)  # experts that have a row, on the average
        return {"bytes": read * 3 * d * f * size + 2 * t * d * size + t * k * 8, "flops": kept * 6 * d * f}
    n, v = case["rows"], case["vocabulary"]
    return {"bytes": n * v * size + n * (16 + 8 * case["top"]), "flops": 6 * n * v}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(state)
    if case["op"] == "mlp":
        return _exact_mlp(state)
    return _exact_logprobs(state)


def _exact_route(s):
    x = s["logits"].double()
    t, e = x.shape
    if s["score"] == "softmax":
        score = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
    else:
        score = torch.sigmoid(x)
    chosen_by = score.clone() if s["bias"] is None else score + s["bias"].double()
    chosen_by[torch.isneginf(x)] = -math.inf
    size = e // s["groups"]
    if s["groups"] > 1:
        strength = torch.full((t, s["groups"]), -math.inf, dtype=torch.float64, device=x.device)
        for g in range(s["groups"]):
            part = chosen_by[:, g * size:(g + 1) * size].clone()
            for _ in range(min(s["group_top"], size)):
                best, at = part.max(1)
                strength[:, g] = torch.where(torch.isneginf(best), strength[:, g],
                                             torch.where(torch.isneginf(strength[:, g]), best, strength[:, g] + best))
                part.scatter_(1, at[:, None], -math.inf)
        rank = (strength[:, None, :] > strength[:, :, None]).sum(2)
        earlier = torch.arange(s["groups"], device=x.device)
        rank += ((strength[:, None, :] == strength[:, :, None]) & (earlier[None, :] < earlier[:, None])).sum(2)
        chosen_by[(rank >= s["top_groups"]).repeat_interleave(size, 1)] = -math.inf
    ids = torch.full((t, s["top_k"]), -1, dtype=torch.int32, device=x.device)
    weights = torch.zeros(t, s["top_k"], dtype=torch.float64, device=x.device)
    places = torch.arange(e, device=x.device).expand(t, e)
    for j in range(s["top_k"]):
        best = chosen_by.max(1, keepdim=True).values
        at = torch.where(chosen_by == best, places, e).min(1, keepdim=True).values
        live = ~torch.isneginf(best)
        ids[:, j:j + 1] = torch.where(live, at, -1).to(torch.int32)
        weights[:, j:j + 1] = torch.where(live, score.gather(1, at), 0.0)
        chosen_by.scatter_(1, at, -math.inf)
    if s["renormalize"]:
        weights = torch.nan_to_num(weights / weights.sum(1, keepdim=True))
    return weights * s["scale"], ids


def _exact_mlp(s):
    x, ids, weights = s["x"].double(), s["ids"], s["weights"].double()
    out = torch.zeros_like(x)
    f = s["inner"]
    for e in range(s["experts"]):
        token, slot = torch.where(ids == e)
        if token.numel():
            both = x[token] @ s["gate_up"][e].double().T
            y = (both[:, :f] * torch.sigmoid(both[:, :f]) * both[:, f:]) @ s["down"][e].double().T
            out.index_add_(0, token, y * weights[token, slot][:, None])
    return out


def _exact_logprobs(s):
    parts = []
    for at in range(0, s["rows"], 256):
        x = s["logits"][at:at + 256].double() * s["scale"]
        rows = x.shape[0]
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(logp)
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
        given = logp[torch.arange(rows, device=x.device), s["tokens"][at:at + 256]]
        values = torch.empty(rows, s["top"], dtype=torch.float64, device=x.device)
        places = torch.empty(rows, s["top"], dtype=torch.int32, device=x.device)
        left = s["logits"][at:at + 256].float().clone()
        places_of = torch.arange(s["vocabulary"], device=x.device)
        for j in range(s["top"]):
            best = left.max(1, keepdim=True).values
            place = torch.where(left == best, places_of, s["vocabulary"]).amin(1, keepdim=True)
            values[:, j:j + 1] = logp.gather(1, place)
            places[:, j:j + 1] = torch.where(torch.isneginf(best), -1, place).to(torch.int32)
            left.scatter_(1, place, -math.inf)
        parts.append((given, entropy, values, places))
    return tuple(torch.cat(column) for column in zip(*parts))
