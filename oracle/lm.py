"""64-bit restatements of the language-model operators (test infrastructure only).

Written row by row from the definitions in include/ttn.h, on CPU tensors.
"""
from __future__ import annotations

import math

import torch


def _ahead(a: float, ia: int, b: float, ib: int) -> bool:
    """NaN first, then the larger, equal values in index order."""
    if math.isnan(a) or math.isnan(b):
        return math.isnan(a) and (not math.isnan(b) or ia < ib)
    return a > b or (a == b and ia < ib)


class _Order:
    def __init__(self, value: float, index: int):
        self.value, self.index = value, index

    def __lt__(self, other):
        return _ahead(self.value, self.index, other.value, other.index)


def _sorted(values, indices):
    return sorted(indices, key=lambda i: _Order(values[i], i))


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, group_top=1, renormalize=False,
          scale=1.0):
    """(weights float64, ids int32, s float64): one row at a time."""
    x = logits.double()
    rows, experts = x.shape
    top_groups = groups if top_groups is None else top_groups
    weights = torch.zeros(rows, top_k, dtype=torch.float64)
    ids = torch.full((rows, top_k), -1, dtype=torch.int32)
    for r in range(rows):
        v = x[r].tolist()
        open_ = [e for e in range(experts) if v[e] != -math.inf]
        if not open_:
            continue
        if score == "softmax":
            if any(math.isnan(v[e]) or v[e] == math.inf for e in open_):
                s = {e: math.nan for e in open_}
            else:
                m = max(v[e] for e in open_)
                total = math.fsum(math.exp(v[e] - m) for e in open_)
                s = {e: math.exp(v[e] - m) / total for e in open_}
        else:
            s = {e: math.nan if math.isnan(v[e]) else 1 / (1 + math.exp(-v[e])) if v[e] > -700 else math.exp(v[e])
                 for e in open_}
        rank = {e: s[e] + (0.0 if bias is None else float(bias[e])) for e in open_}
        if bias is None and (groups == 1 or group_top == 1 or experts == groups):
            # both scores rise with the logit, so its order is the exact one where 64 bits hold the
            # scores no more (0 below -745, 1 above 37)
            rank = {e: rank[e] if math.isnan(rank[e]) else v[e] for e in open_}
        open_ = [e for e in open_ if rank[e] != -math.inf]  # a bias of -inf masks an expert as a logit does
        rank = {e: rank[e] for e in open_}
        if groups > 1:
            size = experts // groups
            strength = []
            for g in range(groups):
                inside = [e for e in open_ if e // size == g]
                best = _sorted(rank, inside)[:group_top]
                strength.append(sum(rank[e] for e in best) if best else -math.inf)
            kept = set(_sorted(strength, range(groups))[:top_groups])
            rank = {e: rank[e] for e in open_ if e // size in kept}
        chosen = _sorted(rank, list(rank))[:top_k]
        w = [s[e] for e in chosen]
        if renormalize:
            total = sum(w)
            w = [0.0 if total == 0 else a / total for a in w]
        for j, e in enumerate(chosen):
            ids[r, j] = e
            weights[r, j] = w[j] * scale
    return weights, ids


def expert_mlp(x, ids, weights, gate_up, down):
    """float64 [tokens, hidden], and a bound on what FP32 accumulation and one rounding of the
    gated activations to x's dtype can move an output before its own rounding."""
    num, hidden, inner = down.shape
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * half  # half a step of subnormal activations
    out = torch.zeros(x.shape, dtype=torch.float64)
    err = torch.zeros(x.shape, dtype=torch.float64)
    f32 = 2.0 ** -24
    for j in range(ids.size(1)):  # in the order of the choices
        for e in range(num):
            t = torch.where(ids[:, j] == e)[0]
            if not len(t):
                continue
            gu, d, v = gate_up[e].double(), down[e].double(), x[t].double()
            both, size = v @ gu.T, v.abs() @ gu.abs().T
            g, u = both[:, :inner], both[:, inner:]
            s = g / (1 + torch.exp(-g))
            h = s * u
            w = weights[t, j].double()[:, None]
            y = h @ d.T
            # a sum of n products: each product and each partial sum rounds once; |silu'| <= 1.1;
            # exp (2 ulp of a value <= 1 + e^-g), the division and the product by u add 8 roundings
            dh = f32 * ((hidden + 2) * (1.1 * size[:, :inner] * u.abs() + s.abs() * size[:, inner:]) + 8 * h.abs())
            dh += half * h.abs() + tiny
            dy = (dh + f32 * (inner + 2) * h.abs()) @ d.abs().T
            out[t] += w * y
            err[t] += w.abs() * dy + f32 * (ids.size(1) + 2) * w.abs() * y.abs()
    return out, err


def token_logprobs(logits, tokens, top=0, scale=1.0):
    """(logprobs, entropy, top_logprobs float64; top_tokens int32)."""
    x = logits.double()
    rows, v = x.shape
    given = torch.zeros(rows, dtype=torch.float64)
    entropy = torch.zeros(rows, dtype=torch.float64)
    values = torch.full((rows, top), -math.inf, dtype=torch.float64)
    places = torch.full((rows, top), -1, dtype=torch.int32)
    for r in range(rows):
        row = x[r]
        live = row != -math.inf
        has = 0 <= int(tokens[r]) < v
        if not bool(live.any()):
            given[r] = -math.inf if has else 0.0
            continue
        bad = bool(torch.isnan(row).any()) or bool((row == math.inf).any())
        if bad:
            logp = torch.full_like(row, math.nan)
            entropy[r] = math.nan
        else:
            z = scale * row
            m = z[live].max()
            logp = z - m - torch.log(torch.exp(z[live] - m).sum())
            entropy[r] = -(torch.exp(logp[live]) * logp[live]).sum()
        if has:
            given[r] = logp[int(tokens[r])]
        if top:
            # NaN first, then larger values; a stable sort keeps index order
            key = torch.where(torch.isnan(row), math.inf, row)
            nan_first = torch.argsort(torch.isnan(row).int(), descending=True, stable=True)
            order = nan_first[torch.argsort(key[nan_first], descending=True, stable=True)]
            if bool((row == math.inf).any()) and bool(torch.isnan(row).any()):
                nans = torch.where(torch.isnan(row))[0]
                order = torch.cat((nans, order[~torch.isnan(row)[order]]))
            order = order[live[order]][:top]
            values[r, :len(order)] = logp[order]
            places[r, :len(order)] = order.int()
            if bad:
                values[r] = math.nan
    return given, entropy, values, places
