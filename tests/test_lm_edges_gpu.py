"""GPU: the language-model operators where magnitudes are far apart or far from one, against
their 64-bit restatements (oracle/lm.py), with the tolerances of test_lm_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import lm
from test_lm_gpu import check_logprobs, check_mlp, check_route, mlp_inputs

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ expert_mlp

@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(60, 96, 64, 4, 2), (300, 96, 64, 3, 1),
                                                                (420, 200, 48, 6, 3), (2400, 72, 2048, 2, 2)])
def test_mlp_features_far_apart_keep_their_own_precision(device, dtype, tokens, hidden, inner, experts, top_k):
    """One output feature in 32 is 10^4 times its neighbours, as massive features of a
    down projection are: the neighbours' error is bounded by their own sums alone."""
    import thintnpu_b200 as ttn
    args = mlp_inputs(tokens, hidden, inner, experts, top_k, DTYPES[dtype], 77)
    args[4][:, 5::32] = (args[4][:, 5::32].double() * 1e4).to(DTYPES[dtype])
    check_mlp(ttn.expert_mlp(*(t.to(device) for t in args)), args)


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("peak", [2.0 ** 125, 2.0 ** 126.5, 3.2e38])
def test_mlp_shares_near_the_largest_float(device, tokens, peak):
    """Shares up to FP32's largest values with routing weights that bring them back.  All
    factors are positive, so no partial sum is larger than its share."""
    import thintnpu_b200 as ttn
    x, ids, weights, gate_up, down = (t.abs() if t.is_floating_point() else t
                                      for t in mlp_inputs(tokens, 64, 32, 3, 2, torch.bfloat16, 19))
    one = torch.ones(tokens, 1)
    largest = max(float(lm.expert_mlp(x, torch.full((tokens, 1), e, dtype=torch.int32), one, gate_up, down)[0].max())
                  for e in range(3))
    # bf16 rounds a factor by 2^-9, the shares' FP32 sums by far less
    down = (down.double() * (peak * (1 - 2.0 ** -6) / largest)).bfloat16()
    args = (x, ids, weights * 2.0 ** -12, gate_up, down)
    got = ttn.expert_mlp(*(t.to(device) for t in args))
    assert bool((got > 0).all())
    check_mlp(got, args)


def test_mlp_calls_of_few_and_many_tiles_in_turn(device):
    """Calls with fewer ring steps than stages, with one tile and with several a CTA pair, close
    behind one another: each is right, repeats itself and leaves no wait unfinished."""
    import thintnpu_b200 as ttn
    sets = [mlp_inputs(tokens, hidden, inner, experts, 1, torch.bfloat16, tokens)
            for tokens, hidden, inner, experts in ((300, 64, 16, 1), (2600, 72, 1024, 2), (270, 520, 48, 9), (9000, 64, 1024, 3))]
    dev = [[t.to(device) for t in args] for args in sets]
    first = [ttn.expert_mlp(*args) for args in dev]
    for _ in range(20):
        again = [ttn.expert_mlp(*args) for args in dev]
    assert ttn.ops.expert_mlp_fault() == 0
    for args, a, b in zip(sets, first, again):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        check_mlp(a, args)


# ------------------------------------------------------------------ route_experts

@pytest.mark.parametrize("size", [3, 4])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("large", [64.0, 1000.0, 1e5])
def test_route_group_sums_of_large_biases_that_cancel(device, size, score, large):
    """A group's two best ranks are near +large and -large: their FP32 sum's error goes with
    the ranks, not with the sum, and group sums differ by less than that."""
    g = torch.Generator().manual_seed(int(large) + size)
    rows, groups = 256, 8
    if score == "sigmoid":
        first = 0.3 + 0.4 * torch.rand(rows, groups, 1, generator=g, dtype=torch.float64)
        second = 1.0 - first + torch.randint(-40, 41, (rows, groups, 1), generator=g) * 2.0 ** -21
        rest = 0.5 * torch.ones(rows, groups, size - 2, dtype=torch.float64)
        s = torch.cat((first, second, rest), 2)
        logits = torch.log(s / (1 - s)).float().view(rows, groups * size)
    else:
        pair = 1.0 / (2 * groups) + torch.randint(-40, 41, (rows, groups, 2), generator=g) * 2.0 ** -22
        rest = 1e-6 * torch.ones(rows, groups, size - 2, dtype=torch.float64)
        logits = torch.log(torch.cat((pair, rest), 2)).float().view(rows, groups * size)
    bias = torch.cat((torch.full((groups, 1), large), torch.full((groups, 1), -large),
                      torch.full((groups, size - 2), -4 * large)), 1).reshape(-1)
    for top_groups in (1, 4):
        check_route(device, logits, 4, score=score, bias=bias, groups=groups, top_groups=top_groups, group_top=2,
                    renormalize=True)


@pytest.mark.parametrize("experts,groups", [(32, 8), (24, 8), (256, 8), (60, 4)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_infinite_biases(device, experts, groups, score):
    """A bias of +inf is an expert that is always wanted, one of -inf an expert that is never
    chosen: its rank is that of a masked expert."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn(9, experts, generator=g)
    logits[1, ::3] = -math.inf
    size = experts // groups
    for wanted, never in (((size + 1,), ()), ((size, size + 1), ()), ((0, experts - 1), (1, size + 2)),
                          ((), tuple(range(size))), ((2,), tuple(range(3, experts)))):
        bias = torch.randn(experts, generator=g) / 10
        bias[list(wanted)] = math.inf
        bias[list(never)] = -math.inf
        check_route(device, logits, 5, score=score, bias=bias)
        for group_top in (1, 2):
            for top_groups in (1, 3):
                check_route(device, logits, 3, score=score, bias=bias, groups=groups, top_groups=top_groups,
                            group_top=group_top, renormalize=True)


@pytest.mark.parametrize("experts", [12, 16])
def test_route_group_sums_beyond_the_largest_float(device, experts):
    """Two ranks of the lowest finite value sum to less than FP32 holds; a group of them is still
    ahead of a group in which everything is masked."""
    groups, size, low = 4, experts // 4, torch.finfo(torch.float32).min
    logits = torch.randn(5, experts, generator=torch.Generator().manual_seed(3))
    logits[:, :size] = -math.inf
    bias = torch.zeros(experts)
    bias[2 * size:] = low
    check_route(device, logits, size + 2, score="sigmoid", bias=bias, groups=groups, top_groups=2, group_top=2)
    bias[2 * size:] = 0.0
    bias[size:2 * size] = -low
    bias[3 * size:] = -low
    check_route(device, logits, 3, score="sigmoid", bias=bias, groups=groups, top_groups=1, group_top=2)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_renormalised_scores_that_all_vanish(device, dtype, groups):
    """Rows under a finite mask of the type's lowest value, or with all chosen logits far below:
    their scores are 0 in 64 bits, and so are the weights (not equal shares)."""
    low = torch.finfo(DTYPES[dtype]).min
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(7, 16, generator=g)
    logits[0] = low
    logits[1, 1:] = low                 # one ordinary expert
    logits[2] = -1000.0 + logits[3]
    logits[4] = -600.0                  # small, but not 0 in 64 bits
    logits[5, 3:] = low
    logits[6] = -math.inf
    logits[6, 5:9] = low
    logits = logits.to(DTYPES[dtype])
    for top_k in (1, 4, 7):
        check_route(device, logits, top_k, score="sigmoid", groups=groups, top_groups=max(1, groups // 2), renormalize=True)
    # a softmax whose chosen experts, wanted by their biases, are far below the row's largest
    logits = torch.randn(4, 16, generator=g)
    logits[:, 4:] -= 60000.0
    logits[1:, 4:] = low
    bias = torch.zeros(16)
    bias[8:] = 2.0
    check_route(device, logits.to(DTYPES[dtype]), 4, score="softmax", bias=bias, groups=groups,
                top_groups=max(1, groups // 2), renormalize=True)


def test_route_refuses_whole_numbers_that_would_wrap(device):
    import thintnpu_b200 as ttn
    logits = torch.randn(3, 16, device=device)
    for kw, message in ((dict(group_top=2 ** 32 + 1), "group_top"), (dict(groups=2 ** 64 + 4, top_groups=2), "groups"),
                        (dict(groups=4, top_groups=2 ** 64 + 1), "top_groups"), (dict(groups=-4), "groups")):
        with pytest.raises(RuntimeError, match=message):
            ttn.route_experts(logits, 2, **kw)


# ------------------------------------------------------------------ token_logprobs

@pytest.mark.parametrize("vocabulary,top", [(40, 8), (5000, 20)])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 21, 1e7, 3e8, 1e9, 1e10, 1e15, 1e20, 1e30, 3e38])
def test_logprobs_far_from_zero(device, size, vocabulary, top):
    """Rows whose largest logit is far from zero on either side, where the scaled maximum has
    no bits left for what separates its neighbours."""
    g = torch.Generator().manual_seed(vocabulary)
    step = size * 2.0 ** -23  # of an FP32 logit
    near = torch.randint(0, 8, (6, vocabulary), generator=g).double() * max(step, 0.5)
    rows = torch.randn(6, vocabulary, generator=g).double()
    rows[0] = -size                                     # everything under a finite mask
    rows[1] = size
    rows[2] = -size - near[2] if size < 1e38 else -size
    rows[3] = size - near[3]
    rows[4, ::7] = size                                 # beside ordinary ones
    rows[5] = -size
    rows[5, 1::9] = -size / 2
    for dtype, scale in (("f32", 1.0), ("f32", 0.3), ("bf16", 1.0)):
        logits = rows.clamp(-3.38e38, 3.38e38).to(DTYPES[dtype])
        check_logprobs(device, logits, torch.randint(vocabulary, (6,), generator=g), top, scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-6, 1e3, 1e6])
def test_logprobs_extreme_scales(device, dtype, scale):
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(6, 3000, generator=g) / min(scale, 1e3)
    rows[1:3] = 60000.0 * torch.randn(2, 3000, generator=g).clamp(-1, 1)
    rows[3] = -54321.0
    rows[4] = 33333.0
    logits = rows.to(DTYPES[dtype])
    check_logprobs(device, logits, torch.randint(3000, (6,), generator=g), 20, scale=scale)


def test_logprobs_differences_beyond_the_largest_float(device):
    """Logits further apart than FP32 holds, brought back into its range by the scale."""
    rows = torch.full((3, 70), 3e38)
    rows[0, 5:] = -3e38
    rows[1, :69] = -2.5e38
    rows[2, ::2] = -3.4e38
    for scale in (1e-6, 0.1, 0.5):
        check_logprobs(device, rows, torch.tensor([60, 3, 4]), 8, scale=scale)
        check_logprobs(device, rows.bfloat16(), torch.tensor([60, 3, 4]), 8, scale=scale)


# ------------------------------------------------------------------ alone and in a batch

def test_a_row_alone_agrees_with_the_row_in_a_batch(device):
    """The number of rows decides the kernels of expert_mlp and the CTAs a row of
    token_logprobs, and a row's address where its vectors begin: values agree within twice the
    bounds that each is held to, the router's bitwise."""
    import thintnpu_b200 as ttn
    g = torch.Generator().manual_seed(23)
    logits = torch.randn(500, 60, generator=g)
    weights, ids = ttn.route_experts(logits.to(device), 4, score="sigmoid", renormalize=True)
    for row in (0, 7, 499):
        w, i = ttn.route_experts(logits[row:row + 1].to(device), 4, score="sigmoid", renormalize=True)
        assert torch.equal(w, weights[row:row + 1]) and torch.equal(i, ids[row:row + 1])

    args = mlp_inputs(300, 200, 96, 5, 2, torch.bfloat16, 29)
    want, err = lm.expert_mlp(*args)
    half = torch.finfo(torch.bfloat16).eps / 2
    bound = 2 * (err + half * (want.abs() + err) + torch.finfo(torch.bfloat16).smallest_normal * half)
    dev = [t.to(device) for t in args]
    batch = ttn.expert_mlp(*dev).cpu().double()
    for rows in (1, 40):
        part = ttn.expert_mlp(*(t[:rows] for t in dev[:3]), *dev[3:]).cpu().double()
        assert bool(((part - batch[:rows]).abs() <= bound[:rows]).all())

    scores = (torch.randn(321, 20011, generator=g) * 3).to(device)  # odd rows: every alignment
    tokens = torch.randint(20011, (321,), generator=g).to(device)
    batch = [t.cpu().double() for t in ttn.token_logprobs(scores, tokens, top=4)]
    for row in (0, 1, 2, 320):
        alone = [t.cpu().double() for t in ttn.token_logprobs(scores[row:row + 1].clone(), tokens[row:row + 1], top=4)]
        assert torch.equal(alone[3], batch[3][row:row + 1])
        for n, (a, b) in enumerate(zip(alone[:3], batch[:3])):
            b = b[row:row + 1]
            z = torch.full_like(b, (math.log(20011) + 1) * (20011 / 256 + 64) / 8) if n == 1 else b.abs() + math.log(20012)
            assert bool(((a - b).abs() <= 2 * (8 * z + 20011 / 256 + 64) * 2.0 ** -24).all())


# ------------------------------------------------------------------ far offsets

def test_offsets_beyond_32_bits(device):
    """Rows 2^31 elements apart, and experts whose weights begin beyond 2^31 elements."""
    import thintnpu_b200 as ttn
    g = torch.Generator().manual_seed(31)
    far = 2 ** 31 + 64
    buffer = torch.zeros(far + 2048, dtype=torch.bfloat16, device=device)

    def spread(rows):  # two rows, far apart
        view = buffer.as_strided((2, rows.size(1)), (far, 1))
        view.copy_(rows)
        return view

    logits = torch.randn(2, 96, generator=g).bfloat16()
    check_route(device, logits, 5, dev_logits=spread(logits), score="sigmoid", renormalize=True)
    scores = torch.randn(2, 1500, generator=g).bfloat16()
    check_logprobs(device, scores, torch.tensor([3, 1499]), 7, dev_logits=spread(scores))

    experts, hidden, inner = 1000, 2048, 544
    used = [0, 510, 998, 999]  # gate_up of the last two begins beyond 2^31 elements
    x, ids, weights, gate_up, down = mlp_inputs(200, hidden, inner, len(used), 2, torch.bfloat16, 37)
    all_gate_up = torch.empty(experts, 2 * inner, hidden, dtype=torch.bfloat16, device=device)
    all_down = torch.empty(experts, hidden, inner, dtype=torch.bfloat16, device=device)
    all_gate_up[used] = gate_up.to(device)
    all_down[used] = down.to(device)
    all_ids = torch.tensor(used, dtype=torch.int32)[ids.long()].to(device)
    for rows in (2, 200):
        got = ttn.expert_mlp(x[:rows].to(device), all_ids[:rows], weights[:rows].to(device), all_gate_up, all_down)
        check_mlp(got, (x[:rows], ids[:rows], weights[:rows], gate_up, down))
    # two tokens far apart, in and out, on the tensor cores: more pairs than the other kernels take
    ids, weights = torch.randint(0, 4, (2, 32), generator=g, dtype=torch.int32), torch.rand(2, 32, generator=g)
    out = torch.zeros(far + 2048, dtype=torch.bfloat16, device=device).as_strided((2, hidden), (far, 1))
    got = ttn.expert_mlp(spread(x[:2]), torch.tensor(used, dtype=torch.int32)[ids.long()].to(device), weights.to(device),
                         all_gate_up, all_down, out=out)
    check_mlp(got, (x[:2], ids, weights, gate_up, down))
