"""CPU: the 64-bit restatements of the language-model operators (oracle/lm.py) against
PyTorch's own operations where those define the same thing."""
from __future__ import annotations

import math

import torch

from oracle import lm


def test_route_is_topk_of_softmax_and_sigmoid():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20, 40, generator=g)
    for score, s in (("softmax", torch.softmax(x.double(), 1)), ("sigmoid", torch.sigmoid(x.double()))):
        weights, ids = lm.route(x, 6, score=score, scale=2.0)
        top = torch.topk(s, 6, dim=1)
        assert torch.equal(ids.long(), top.indices)
        assert torch.allclose(weights, 2 * top.values, rtol=1e-14, atol=0)
        bias = torch.randn(40, generator=g)
        weights, ids = lm.route(x, 6, score=score, bias=bias, renormalize=True)
        top = torch.topk(s + bias.double(), 6, dim=1)
        assert torch.equal(ids.long(), top.indices)
        chosen = s.gather(1, top.indices)
        assert torch.allclose(weights, chosen / chosen.sum(1, keepdim=True), rtol=1e-13, atol=0)


def test_route_groups_masks_and_ties():
    x = torch.tensor([[1.0, 5.0, 4.0, 4.5, 0.0, 3.0, 2.0, 2.5]])
    # sigmoid sums of the two best: (5, 1), (4.5, 4), (3, 0), (2.5, 2); the best: 5, 4.5, 3, 2.5
    assert lm.route(x, 3, score="sigmoid", groups=4, top_groups=1, group_top=2)[1].tolist() == [[3, 2, -1]]
    assert lm.route(x, 3, score="sigmoid", groups=4, top_groups=2, group_top=1)[1].tolist() == [[1, 3, 2]]
    tied = torch.zeros(1, 6)
    assert lm.route(tied, 3)[1].tolist() == [[0, 1, 2]]
    tied[0, :2] = -math.inf
    weights, ids = lm.route(tied, 6, renormalize=True)
    assert ids.tolist() == [[2, 3, 4, 5, -1, -1]] and weights[0, 4:].tolist() == [0, 0]
    nan = torch.tensor([[0.0, math.nan, 1.0]])
    assert lm.route(nan, 2, score="sigmoid")[1].tolist() == [[1, 2]]
    assert lm.route(nan, 2, score="softmax")[1].tolist() == [[0, 1]]  # every score is NaN


def test_expert_mlp_is_the_sum_of_gated_products():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 8, generator=g).bfloat16()
    ids = torch.tensor([[0, 1], [1, 1], [-1, 0], [2, 9], [7, -5]], dtype=torch.int32)
    w = torch.rand(5, 2, generator=g)
    gate_up, down = torch.randn(3, 32, 8, generator=g).bfloat16(), torch.randn(3, 8, 16, generator=g).bfloat16()
    out, err = lm.expert_mlp(x, ids, w, gate_up, down)
    for t in range(5):
        want = torch.zeros(8, dtype=torch.float64)
        for j in range(2):
            e = int(ids[t, j])
            if 0 <= e < 3:
                both = gate_up[e].double() @ x[t].double()
                want += float(w[t, j]) * (down[e].double() @ (torch.nn.functional.silu(both[:16]) * both[16:]))
        assert torch.allclose(out[t], want, rtol=1e-12, atol=1e-12)
    assert bool((out[4] == 0).all()) and bool((err[4] == 0).all()) and bool((err[:4] > 0).all())


def test_token_logprobs_are_log_softmax():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 50, generator=g)
    x[1, 10:40] = -math.inf
    tokens = torch.tensor([0, 3, 49, -1, 50, 7])
    given, entropy, values, places = lm.token_logprobs(x, tokens, 5, scale=1.5)
    logp = torch.log_softmax(x.double() * 1.5, 1)
    for r, t in enumerate(tokens.tolist()):
        assert given[r] == 0 if not 0 <= t < 50 else torch.allclose(given[r], logp[r, t], rtol=1e-13)
    p = torch.where(logp == -math.inf, 0.0, logp.exp() * logp)
    assert torch.allclose(entropy, -p.sum(1), rtol=1e-12)
    top = torch.topk(logp, 5, dim=1)
    assert torch.equal(places.long(), top.indices) and torch.allclose(values, top.values, rtol=1e-13)
    few = torch.full((1, 4), -math.inf)
    few[0, 2] = 1.0
    given, entropy, values, places = lm.token_logprobs(few, torch.tensor([0]), 3)
    assert places.tolist() == [[2, -1, -1]] and values[0].tolist() == [0.0, -math.inf, -math.inf]
    assert given.tolist() == [-math.inf] and entropy.tolist() == [0.0]
