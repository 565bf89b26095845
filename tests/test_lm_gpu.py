"""GPU parity of the language-model operators (route_experts, expert_mlp,
token_logprobs) with their 64-bit restatements (oracle/lm.py).

Tolerances are derived, not tuned.  With u = 2^-24 (half an FP32 step, relative):
* route weights: numerator and denominator exponentials are within 2 ulp (8 u in all),
  each argument x - max is rounded (|x - max| u, twice), at most 32 + 5 additions form a
  row's sum and 16 + 5 a renormalised one, and six more operations round once:
  (80 + 2 range) u relative.  Chosen experts and their order must be equal.
* log probabilities: z = scale (x - max) rounds twice, log S and the difference once, S is a sum
  whose terms carry 2^-22 (exp2) and |z| u, accumulated in at most n / 256 + 24 steps:
  (8 |z| + n / 256 + 64) u absolute; top tokens must be equal.
* expert_mlp: the bound that the oracle adds up term by term, plus the output's rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


# ------------------------------------------------------------------ route_experts

def check_route(device, logits, top_k, dev_logits=None, **kw):
    import thintnpu_b200 as ttn
    dev_kw = dict(kw)
    if kw.get("bias") is not None:
        dev_kw["bias"] = kw["bias"].to(device)
    weights, ids = ttn.route_experts(logits.to(device) if dev_logits is None else dev_logits, top_k, **dev_kw)
    want_w, want_ids = lm.route(logits, top_k, **kw)
    assert weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_ids)
    got = weights.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want_w))
    # the lowest finite value has a score of 0 in any precision
    fine = torch.isfinite(logits) & (logits > torch.finfo(logits.dtype).min)
    x = logits.double()
    spread = torch.where(fine, x, -math.inf).amax(1, keepdim=True) - torch.where(fine, x, math.inf).amin(1, keepdim=True)
    spread = torch.where(torch.isfinite(spread), spread, 0.0)
    live = ~torch.isnan(want_w)
    # FP32's smallest normal: below it weights lose relative precision
    bound = (80 + 2 * spread) * U * want_w.abs() + 2.0 ** -126
    assert bool(((got - want_w).abs() <= bound)[live].all()), float(((got - want_w).abs() - bound)[live].max())


ROUTE = [  # rows, experts, top_k, groups, top_groups
    (1, 1, 1, 1, 1), (1, 2, 2, 1, 1), (5, 8, 2, 1, 1), (33, 31, 5, 1, 1), (7, 33, 8, 1, 1), (64, 64, 8, 1, 1),
    (9, 64, 4, 8, 3), (17, 60, 6, 4, 2), (40, 160, 6, 8, 3), (50, 256, 8, 8, 4), (3, 255, 16, 5, 2), (4, 512, 10, 16, 7),
    (3, 1024, 16, 32, 9), (6, 96, 3, 32, 5), (11, 128, 16, 1, 1), (5, 16, 16, 4, 3), (8, 9, 9, 9, 4)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased,group_top,renormalize", [(False, 1, True), (True, 2, True), (True, 1, False),
                                                          (False, 2, False)])
def test_route_sizes(device, dtype, score, biased, group_top, renormalize):
    for n, (rows, experts, top_k, groups, top_groups) in enumerate(ROUTE):
        g = torch.Generator().manual_seed(100 + n)
        logits = (torch.randn(rows, experts, generator=g) * 2).to(DTYPES[dtype])
        bias = torch.round(torch.randn(experts, generator=g) * 50) / 1000 if biased else None
        check_route(device, logits, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                    group_top=group_top, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masks_ties_and_nonfinite(device, score, biased, groups):
    g = torch.Generator().manual_seed(7)
    experts = 24
    rows = torch.randn(12, experts, generator=g)
    rows[0] = -math.inf                       # nothing left
    rows[1, 1:] = -math.inf                   # one left
    rows[2, 3:] = -math.inf                   # fewer than top_k left
    rows[3] = 0.5                             # all tied
    rows[4, ::2] = 1.25                       # ties between groups
    rows[5] = torch.finfo(torch.float32).min  # the lowest value is a number, not a mask
    rows[6, :20] = torch.finfo(torch.float32).min
    rows[7, 5] = math.nan
    rows[8, 9] = math.inf
    rows[9, 2], rows[9, 11], rows[9, 12:] = math.nan, math.nan, -math.inf
    rows[10] = -0.0
    rows[10, ::3] = 0.0                       # equal to -0
    bias = torch.round(torch.randn(experts, generator=g) * 10) / 100 if biased else None
    if biased:
        bias[4:8] = bias[0:4]
    for group_top in (1, 2):
        for renormalize in (False, True):
            if score == "sigmoid" and renormalize:
                rows[5:7] = rows[11]  # sums of scores that all vanish in 64 bits too have no value to compare
            for top_k in (1, 6, 16):
                check_route(device, rows, top_k, score=score, bias=bias, groups=groups,
                            top_groups=max(1, groups // 2), group_top=group_top, renormalize=renormalize)


def test_route_close_ranks_are_ordered_exactly(device):
    """Ranks closer than FP32 resolves: logits a few steps apart around the choice, biases
    that nearly undo the difference of the scores, and group sums that nearly tie."""
    g = torch.Generator().manual_seed(11)
    for score in ("softmax", "sigmoid"):
        for rows, experts, top_k in ((64, 64, 8), (16, 200, 16), (32, 40, 3)):
            base = torch.full((rows, experts), 0.75) + torch.randint(-6, 7, (rows, experts), generator=g) * 2.0 ** -23
            check_route(device, base, top_k, score=score, bias=torch.zeros(experts))
            check_route(device, base, top_k, score=score)
            # rank = s + b with b = c - s rounded to FP32: all ranks within a few roundings of c
            x = torch.randn(1, experts, generator=g).repeat(rows, 1)
            s = torch.softmax(x.double(), 1) if score == "softmax" else torch.sigmoid(x.double())
            bias = (0.6 - s[0]).float()
            check_route(device, x, top_k, score=score, bias=bias, renormalize=True)
            check_route(device, x, top_k, score=score, bias=bias, groups=4, top_groups=2, group_top=2)


def test_route_close_ranks_of_many_experts(device):
    """1024 softmax scores and biases that undo their differences to a few roundings."""
    g = torch.Generator().manual_seed(13)
    x = (torch.randn(1, 1024, generator=g) * 4).repeat(6, 1)
    s = torch.softmax(x.double(), 1)
    bias = (0.5 - s[0]).float()
    bias += torch.randint(-30, 31, (1024,), generator=g) * 2.0 ** -24
    check_route(device, x, 16, bias=bias)
    check_route(device, x, 16, bias=bias, groups=32, top_groups=7, group_top=2, renormalize=True)


def test_route_small_sigmoids_keep_their_ratios(device):
    logits = torch.tensor([[-90.0, -91.0, -95.0, -130.0], [-19.5, -20.5, -21.0, -200.0]])
    check_route(device, logits, 3, score="sigmoid", renormalize=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_route_strides_and_offsets(device, dtype):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(40, 3, 300, generator=g).to(DTYPES[dtype])
    dev = big.to(device)
    for cut in (lambda t: t[:, 1, 7:263], lambda t: t[:, 0, 8:264], lambda t: t[3:, 2, ::2][:, :96],
                lambda t: t[:, :, 5], lambda t: t[:20, 0, :64].t(), lambda t: t[0, :, :128].expand(3, 128)):
        check_route(device, cut(big), 3, dev_logits=cut(dev), score="sigmoid", renormalize=True)
    row = big[:1, 0, :64].expand(9, 64)  # a row stride of zero
    check_route(device, row, 4, dev_logits=dev[:1, 0, :64].expand(9, 64))


def test_route_outputs_and_empty(device):
    import thintnpu_b200 as ttn
    logits = torch.randn(6, 32, generator=torch.Generator().manual_seed(1))
    weights = torch.full((8, 4), 7.0, device=device)
    ids = torch.full((8, 4), 7, dtype=torch.int32, device=device)
    ttn.route_experts(logits.to(device), 4, out=(weights[:6], ids[:6]))
    want_w, want_ids = lm.route(logits, 4)
    assert torch.equal(ids[:6].cpu(), want_ids)
    assert bool((weights[6:] == 7).all()) and bool((ids[6:] == 7).all())  # rows behind the last stay
    w, i = ttn.route_experts(torch.empty(0, 32, device=device), 4)
    assert w.shape == (0, 4) and i.shape == (0, 4)


# ------------------------------------------------------------------ expert_mlp

def mlp_inputs(tokens, hidden, inner, experts, top_k, dtype, seed, dropped=0.0, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g).to(dtype)
    scores = torch.randn(tokens, experts, generator=g) + skew * torch.arange(experts)
    ids = torch.topk(scores, top_k, dim=1).indices.to(torch.int32)
    if dropped:
        ids[torch.rand(tokens, top_k, generator=g) < dropped] = -1
    weights = torch.rand(tokens, top_k, generator=g)
    gate_up = (torch.randn(experts, 2 * inner, hidden, generator=g) * hidden ** -0.5).to(dtype)
    down = (torch.randn(experts, hidden, inner, generator=g) * inner ** -0.5).to(dtype)
    return x, ids, weights, gate_up, down


def check_mlp(got, args):
    want, err = lm.expert_mlp(*args)
    dtype = args[0].dtype
    half = torch.finfo(dtype).eps / 2
    bound = err + half * (want.abs() + err) + torch.finfo(dtype).smallest_normal * half
    far = (got.cpu().double() - want).abs() - bound
    assert got.dtype == dtype and bool((far <= 0).all()), float(far.max())


MLP = [  # tokens, hidden, inner, experts, top_k, dropped, skew
    (1, 8, 16, 1, 1, 0.0, 0.0), (1, 64, 48, 4, 2, 0.0, 0.0), (1, 136, 80, 8, 8, 0.0, 0.0), (3, 256, 128, 5, 3, 0.3, 0.0),
    (2, 1032, 688, 4, 2, 0.0, 0.0), (17, 72, 16, 7, 1, 0.0, 0.0), (40, 264, 112, 6, 4, 0.25, 0.0),
    (129, 64, 64, 3, 2, 0.0, 0.5), (300, 128, 144, 2, 2, 0.1, 0.0), (65, 520, 272, 40, 6, 0.0, 0.05),
    (600, 40, 32, 4, 3, 0.0, 1.0), (33, 512, 256, 2, 1, 0.0, 3.0), (260, 328, 208, 1, 1, 0.0, 0.0),
    # more than 256 pairs: on the tensor cores, down to the smallest sizes
    (300, 8, 16, 1, 1, 0.0, 0.0), (280, 1032, 688, 4, 2, 0.1, 0.0), (90, 264, 112, 6, 4, 0.25, 0.0),
    (257, 64, 48, 64, 1, 0.0, 0.0), (34, 512, 256, 3, 1, 0.0, 0.0), (20, 2048, 1024, 3, 1, 0.0, 0.0),
    # the most experts and the most choices
    (400, 16, 16, 1024, 2, 0.0, 0.0), (1200, 24, 32, 1024, 2, 0.1, 0.0), (40, 40, 16, 64, 32, 0.3, 0.0),
    (1, 64, 32, 40, 32, 0.1, 0.0),
    # many rows an expert: two sub-tiles in the first product, in the second, in both with ragged runs
    (2400, 72, 2048, 2, 2, 0.0, 0.3), (4760, 2048, 48, 3, 2, 0.1, 0.4), (5000, 1000, 992, 5, 2, 0.05, 0.2)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k,dropped,skew", MLP)
def test_mlp_sizes(device, dtype, tokens, hidden, inner, experts, top_k, dropped, skew):
    import thintnpu_b200 as ttn
    args = mlp_inputs(tokens, hidden, inner, experts, top_k, DTYPES[dtype], tokens + hidden, dropped, skew)
    check_mlp(ttn.expert_mlp(*(t.to(device) for t in args)), args)


@pytest.mark.parametrize("tokens", [2, 90, 200])
def test_mlp_strided_rows_and_output(device, tokens):
    import thintnpu_b200 as ttn
    args = mlp_inputs(tokens, 96, 32, 4, 2, torch.bfloat16, 5)
    x, ids, weights, gate_up, down = (t.to(device) for t in args)
    wide = torch.zeros(tokens, 3, 104, dtype=torch.bfloat16, device=device)
    wide[:, 1, :96] = x
    out = torch.full((tokens + 2, 2, 96), 5.0, dtype=torch.bfloat16, device=device)
    got = ttn.expert_mlp(wide[:, 1, :96], ids, weights, gate_up, down, out=out[:tokens, 1])
    check_mlp(got, args)
    assert bool((out[:, 0] == 5).all()) and bool((out[tokens:] == 5).all())


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_mlp_tokens_without_experts(device, tokens):
    """Ids outside the experts (no choice, another rank's expert) add nothing, even with
    NaN weights; a token with no other id gets zeros; an empty call does nothing."""
    import thintnpu_b200 as ttn
    args = list(mlp_inputs(tokens, 64, 32, 4, 3, torch.float16, 9))
    args[1][0] = torch.tensor([-1, 4, 2 ** 31 - 1], dtype=torch.int32)
    args[1][-1, 0] = -2 ** 31
    args[2][0] = math.nan
    args[2][-1, 0] = math.inf
    got = ttn.expert_mlp(*(t.to(device) for t in args))
    if tokens > 1:
        assert bool((got[0] == 0).all())
    args[2][0] = 0.0
    args[2][-1, 0] = 0.0
    check_mlp(got, args)
    all_out = torch.full_like(args[1], -1)
    assert bool((ttn.expert_mlp(args[0].to(device), all_out.to(device), *(t.to(device) for t in args[2:])) == 0).all())
    x, _, _, gate_up, down = (t.to(device) for t in args)
    none = ttn.expert_mlp(x[:0], all_out[:0].to(device), args[2][:0].to(device), gate_up, down)
    assert none.shape == (0, 64)


@pytest.mark.parametrize("tokens", [2, 150])
def test_mlp_same_expert_twice_and_nonfinite(device, tokens):
    import thintnpu_b200 as ttn
    args = list(mlp_inputs(tokens, 64, 32, 3, 2, torch.bfloat16, 21))
    args[1][:, 1] = args[1][:, 0]
    check_mlp(ttn.expert_mlp(*(t.to(device) for t in args)), args)
    args[0][0, 3] = math.nan  # one token's NaN stays with it
    got = ttn.expert_mlp(*(t.to(device) for t in args))
    assert bool(torch.isnan(got[0]).all()) and not bool(torch.isnan(got[1:]).any())
    args[0][0, 3] = 0.0
    args[2][0, 0] = math.inf
    got = ttn.expert_mlp(*(t.to(device) for t in args)).cpu().double()
    plain, _ = lm.expert_mlp(*args)
    sure = plain[0].abs() == math.inf
    assert torch.equal(got[0][sure], plain[0][sure])
    assert bool(torch.isfinite(got[1:]).all())


def test_mlp_is_deterministic_and_order_free(device):
    """The same call gives the same bits, and a token's result does not depend on the
    other tokens' order beyond the tile it falls into: bitwise equal for a permuted batch."""
    import thintnpu_b200 as ttn
    args = [t.to(device) for t in mlp_inputs(500, 128, 64, 6, 3, torch.bfloat16, 2)]
    first = ttn.expert_mlp(*args)
    assert torch.equal(first.view(torch.int16), ttn.expert_mlp(*args).view(torch.int16))
    perm = torch.randperm(500, generator=torch.Generator().manual_seed(4)).to(device)
    moved = ttn.expert_mlp(args[0][perm].contiguous(), args[1][perm].contiguous(), args[2][perm].contiguous(), *args[3:])
    assert torch.equal(first[perm].view(torch.int16), moved.view(torch.int16))


@pytest.mark.parametrize("tokens", [5, 130])
def test_mlp_given_workspace_and_odd_addresses(device, tokens):
    """Ids and weights at addresses that are only 4-byte aligned, and a workspace of the
    caller's, larger than needed and dirty."""
    import thintnpu_b200 as ttn
    args = mlp_inputs(tokens, 96, 48, 5, 3, torch.bfloat16, 31, dropped=0.1)
    x, ids, weights, gate_up, down = (t.to(device) for t in args)
    odd_ids = torch.empty(tokens * 3 + 1, dtype=torch.int32, device=device)[1:].view(tokens, 3)
    odd_weights = torch.empty(tokens * 3 + 1, device=device)[1:].view(tokens, 3)
    odd_ids.copy_(ids)
    odd_weights.copy_(weights)
    need = ttn.ops.expert_mlp_workspace_size(tokens, 96, 48, 5, 3)
    workspace = torch.full((need + 512,), 255, dtype=torch.uint8, device=device)
    for _ in range(2):
        check_mlp(ttn.expert_mlp(x, odd_ids, odd_weights, gate_up, down, workspace=workspace), args)
    assert bool((workspace[need:] == 255).all())


def test_mlp_two_streams_at_once(device):
    import thintnpu_b200 as ttn
    sets = [[t.to(device) for t in mlp_inputs(700, 256, 128, 6, 2, torch.float16, seed)] for seed in (1, 2)]
    want = [ttn.expert_mlp(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(ttn.expert_mlp(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g.view(torch.int16), want[i].view(torch.int16))
    assert ttn.ops.expert_mlp_fault() == 0


def test_mlp_bounded_waits_run_out_and_the_next_call_is_right(device):
    """A call whose first product gets no operands gives up within its limits and says why;
    the context and the next call are unharmed."""
    import thintnpu_b200 as ttn
    from thintnpu_b200 import _lib
    args = mlp_inputs(200, 128, 64, 4, 2, torch.bfloat16, 3)
    dev = [t.to(device) for t in args]
    assert ttn.ops.expert_mlp_fault() == 0
    _lib.lib().ttn_expert_mlp_test_withhold_copies()
    ttn.expert_mlp(*dev)
    torch.cuda.synchronize()
    assert ttn.ops.expert_mlp_fault() == 5
    check_mlp(ttn.expert_mlp(*dev), args)
    assert ttn.ops.expert_mlp_fault() == 0


# ------------------------------------------------------------------ token_logprobs

def check_logprobs(device, logits, tokens, top, scale=1.0, dev_logits=None):
    import thintnpu_b200 as ttn
    got = ttn.token_logprobs(logits.to(device) if dev_logits is None else dev_logits, tokens.to(device), top=top,
                             scale=scale)
    given, entropy, values, places = (t.cpu() for t in got)
    want = lm.token_logprobs(logits, tokens, top, scale)
    assert torch.equal(places, want[3])
    n = logits.size(1)

    def near(a, b, size):
        # 2 * -FLT_MAX = -6.8e38 lies beyond FP32's range (2^128 = 3.4e38): its FP32 value is -inf
        a, b = a.double(), b.float().double()
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        fine = torch.isfinite(b)
        far = ((a - b).abs() - (8 * size + n / 256 + 64) * U)[fine]
        assert not far.numel() or float(far.max()) <= 0, float(far.max())

    z = want[0].abs() + math.log(n + 1)  # |scale (x - max)| <= |log p| + log S
    near(given, want[0], z)
    # A / S = sum p |z|: each term as a log probability's; |z| of the terms that count is
    # weighed by p, and sum p |z| <= entropy <= log n
    near(entropy, want[1], torch.full_like(want[1], (math.log(n) + 1) * (n / 256 + 64) / 8))
    near(values, want[2], want[2].abs() + math.log(n + 1))


LOGPROBS = [(1, 1, 1), (1, 2, 1), (3, 7, 3), (2, 31, 20), (5, 255, 5), (4, 256, 32), (3, 257, 20), (2, 1000, 0),
            (2, 4097, 20), (1, 32003, 20), (200, 513, 2), (1, 131073, 32)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocabulary,top", LOGPROBS)
def test_logprobs_sizes(device, dtype, rows, vocabulary, top):
    g = torch.Generator().manual_seed(rows + vocabulary)
    logits = (torch.randn(rows, vocabulary, generator=g) * 3).to(DTYPES[dtype])
    tokens = torch.randint(vocabulary, (rows,), generator=g)
    check_logprobs(device, logits, tokens, top)
    check_logprobs(device, logits, tokens, top, scale=0.7)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocabulary,top", [(40, 8), (3000, 20)])
def test_logprobs_masks_ties_and_nonfinite(device, dtype, vocabulary, top):
    g = torch.Generator().manual_seed(5)
    low = torch.finfo(DTYPES[dtype]).min
    rows = torch.randn(16, vocabulary, generator=g)
    rows[0] = -math.inf                               # nothing left
    rows[1, 1:] = -math.inf                           # one left
    rows[2, torch.rand(vocabulary, generator=g) < 0.9] = -math.inf
    rows[3] = 0.25                                    # all tied
    rows[4, vocabulary // 3:] = 2.5                   # a long tie at the top
    rows[5] = low
    rows[6, 1:] = low
    rows[7, vocabulary // 2] = math.nan
    rows[8, 3] = math.inf
    rows[9, 5], rows[9, 6], rows[9, 7:] = math.nan, math.inf, -math.inf
    rows[10] = torch.arange(vocabulary) / 16.0        # every element beats all before it
    rows[11] = -torch.arange(vocabulary) / 16.0
    rows[12] = -0.0
    rows[12, 1::2] = 0.0
    rows[13] = 1000.0 + rows[14]                      # far from zero
    logits = rows.to(DTYPES[dtype])
    tokens = torch.randint(vocabulary, (16,), generator=g)
    tokens[1] = 0
    tokens[2] = -100          # a row without a given token
    tokens[3] = vocabulary    # outside
    tokens[4] = 2 ** 40
    check_logprobs(device, logits, tokens, top)
    check_logprobs(device, logits, tokens, 0, scale=2.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_logprobs_strides_and_offsets(device, dtype):
    g = torch.Generator().manual_seed(6)
    big = (torch.randn(6, 2, 1303, generator=g) * 2).to(DTYPES[dtype])
    dev = big.to(device)
    tokens = torch.randint(600, (6,), generator=g)
    for cut in (lambda t: t[:, 1, 1:1001], lambda t: t[:, 0, 3:700], lambda t: t[:, 1], lambda t: t[:, 0, 5:1303]):
        check_logprobs(device, cut(big), tokens, 6, dev_logits=cut(dev))
    check_logprobs(device, big[2:3, 0].expand(6, -1), tokens, 3, dev_logits=dev[2:3, 0].expand(6, -1))


def test_logprobs_large_vocabulary_and_empty(device):
    import thintnpu_b200 as ttn
    g = torch.Generator().manual_seed(8)
    logits = (torch.randn(2, 1 << 20, generator=g) * 2).to(torch.bfloat16)
    check_logprobs(device, logits, torch.tensor([5, (1 << 20) - 1]), 32)
    out = ttn.token_logprobs(torch.empty(0, 100, device=device), torch.empty(0, dtype=torch.int64, device=device), top=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logprobs_few_left_and_equal_rows(device, dtype):
    """Rows under a narrow mask (fewer tokens left than the alternatives asked for, spread over
    the vocabulary), constant rows, and rows that rise or fall by the finest steps."""
    g = torch.Generator().manual_seed(12)
    v = 20011
    rows = torch.full((8, v), -math.inf)
    for r, left in ((0, 3), (1, 40)):
        at = torch.randperm(v, generator=g)[:left]
        rows[r, at] = torch.randn(left, generator=g)
    rows[2] = 0.0
    rows[3] = torch.finfo(DTYPES[dtype]).min
    rows[4, ::2] = 1.5
    rows[5] = torch.arange(v) * 2.0 ** -10
    rows[6] = torch.arange(v).flip(0) * 2.0 ** -10
    rows[7, -1] = -2.0
    tokens = torch.randint(v, (8,), generator=g)
    for top in (1, 20, 32):
        check_logprobs(device, rows.to(DTYPES[dtype]), tokens, top)


def test_logprobs_many_rows_of_the_largest_vocabulary(device):
    """One CTA a row holds every segment maximum of a 2^20 vocabulary: more than 48 KB of
    shared memory (the rows are one row, expanded)."""
    import thintnpu_b200 as ttn
    g = torch.Generator().manual_seed(14)
    row = (torch.randn(1, 1 << 20, generator=g) * 2).float()
    want = lm.token_logprobs(row, torch.tensor([77]), 20)
    got = ttn.token_logprobs(row.to(device).expand(400, -1), torch.full((400,), 77).to(device), top=20)
    assert torch.equal(got[3].cpu(), want[3].expand(400, -1))
    bound = (8 * (want[2].abs() + math.log(1 << 20)) + (1 << 20) / 256 + 64) * U
    assert bool(((got[2].cpu().double() - want[2]).abs() <= bound).all())
    assert torch.equal(got[0], got[0][:1].expand(400))


# ------------------------------------------------------------------ together

def _layer(ttn, x, router, bias, gate_up, down, head, tokens):
    """A mixture-of-experts layer with a residual, then the read-out of given tokens."""
    logits = x.float() @ router
    weights, ids = ttn.route_experts(logits, 2, score="sigmoid", bias=bias, groups=2, top_groups=1, group_top=2,
                                     renormalize=True)
    y = x + ttn.expert_mlp(x, ids, weights, gate_up, down)
    return ttn.token_logprobs(y @ head, tokens, top=3) + (ids, weights, y)


@pytest.mark.parametrize("tokens", [1, 5, 130])
def test_layer_and_read_out_eager_captured_and_on_another_stream(device, tokens):
    import thintnpu_b200 as ttn
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, 64, generator=g).bfloat16().to(device)
    router = torch.randn(64, 8, generator=g).to(device) / 8
    bias = (torch.randn(8, generator=g) / 10).to(device)
    gate_up = (torch.randn(8, 96, 64, generator=g) / 8).bfloat16().to(device)
    down = (torch.randn(8, 64, 48, generator=g) / 7).bfloat16().to(device)
    head = (torch.randn(64, 500, generator=g) / 4).bfloat16().to(device)
    given = torch.randint(500, (tokens,), generator=g).to(device)
    args = (router, bias, gate_up, down, head, given)
    eager = _layer(ttn, x, *args)

    logits = (x.float() @ router).cpu()
    want_w, want_ids = lm.route(logits, 2, score="sigmoid", bias=bias.cpu(), groups=2, top_groups=1, group_top=2,
                                renormalize=True)
    assert torch.equal(eager[4].cpu(), want_ids)
    out = ttn.expert_mlp(x, eager[4], eager[5], gate_up, down)
    assert ttn.ops.expert_mlp_fault() == 0
    check_mlp(out, tuple(t.cpu() for t in (x, eager[4], eager[5], gate_up, down)))
    check_logprobs(device, (eager[6] @ head).cpu(), given.cpu(), 3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(_layer(ttn, x, *args), eager):
            assert torch.equal(a, b)
        graphs, held = [], []
        for _ in range(2):  # two graphs, replayed in turn: each has its own workspace
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held.append(_layer(ttn, x, *args))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        new = torch.randn(tokens, 64, generator=g).bfloat16().to(device)
        x.copy_(new)
        for graph in graphs:
            graph.replay()
        fresh = _layer(ttn, x, *args)
        for graph_out in held:
            for a, b in zip(graph_out, fresh):
                assert torch.equal(a, b), step


def test_operators_through_torch_ops(device):
    import thintnpu_b200 as ttn
    from thintnpu_b200 import library  # noqa: F401
    g = torch.Generator().manual_seed(1)
    nf = torch.ops.thin_native_flow
    logits = torch.randn(4, 16, generator=g).to(device)
    w, ids = nf.route_experts(logits, 2, "sigmoid", None, 4, 2, 2, True, 1.5)
    w2, ids2 = ttn.route_experts(logits, 2, score="sigmoid", groups=4, top_groups=2, group_top=2, renormalize=True,
                                 scale=1.5)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    x = torch.randn(4, 32, generator=g).half().to(device)
    gate_up, down = torch.randn(16, 64, 32, generator=g).half().to(device), torch.randn(16, 32, 32, generator=g).half().to(device)
    assert torch.equal(nf.expert_mlp(x, ids, w, gate_up, down), ttn.expert_mlp(x, ids, w, gate_up, down))
    tokens = torch.tensor([1, 2, 3, 4]).to(device)
    for a, b in zip(nf.token_logprobs(logits, tokens, 3, 1.0), ttn.token_logprobs(logits, tokens, top=3)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ refusals

def test_refusals(device):
    import thintnpu_b200 as ttn
    logits = torch.randn(4, 16, device=device)
    bad = [
        (lambda: ttn.route_experts(logits.double(), 2), "dtype"),
        (lambda: ttn.route_experts(logits[0], 2), "rows, columns"),
        (lambda: ttn.route_experts(logits.cpu(), 2), "CUDA"),
        (lambda: ttn.route_experts(logits, 0), "top_k"),
        (lambda: ttn.route_experts(logits, 17), "top_k"),
        (lambda: ttn.route_experts(torch.randn(2, 64, device=device), 17), "top_k"),
        (lambda: ttn.route_experts(torch.randn(2, 1025, device=device), 2), "1024"),
        (lambda: ttn.route_experts(logits, 2, score="relu"), "score"),
        (lambda: ttn.route_experts(logits, 2, groups=3), "groups"),
        (lambda: ttn.route_experts(logits, 2, groups=4, top_groups=5), "top_groups"),
        (lambda: ttn.route_experts(logits, 2, groups=4, top_groups=2, group_top=3), "group_top"),
        (lambda: ttn.route_experts(logits, 2, bias=torch.zeros(16, device=device).half()), "bias"),
        (lambda: ttn.route_experts(logits, 2, bias=torch.zeros(15, device=device)), "bias"),
        (lambda: ttn.route_experts(logits, 2, scale=math.nan), "scale"),
        (lambda: ttn.route_experts(logits, 2, scale=math.inf), "scale"),
        (lambda: ttn.route_experts(logits.requires_grad_(), 2), "inference-only"),
    ]
    x = torch.randn(4, 32, device=device).half()
    ids, w = torch.zeros(4, 2, dtype=torch.int32, device=device), torch.ones(4, 2, device=device)
    gate_up, down = torch.randn(3, 64, 32, device=device).half(), torch.randn(3, 32, 32, device=device).half()
    bad += [
        (lambda: ttn.expert_mlp(x.float(), ids, w, gate_up, down), "float16"),
        (lambda: ttn.expert_mlp(x, ids.long(), w, gate_up, down), "experts"),
        (lambda: ttn.expert_mlp(x, ids[:3], w, gate_up, down), "experts"),
        (lambda: ttn.expert_mlp(x, ids, w.half(), gate_up, down), "weights"),
        (lambda: ttn.expert_mlp(x, ids, w[:, :1], gate_up, down), "weights"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up.bfloat16(), down), "gate_up"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up[:, :63], down), "gate_up"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up, down[:2]), "down"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up, down.transpose(1, 2)), "down"),
        (lambda: ttn.expert_mlp(x[:, :28], ids, w, gate_up[:, :, :28].contiguous(), down[:, :28].contiguous()), "multiple of 8"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up[:, :48].contiguous(), down[:, :, :24].contiguous()), "16"),
        (lambda: ttn.expert_mlp(torch.randn(32, 4, device=device).half().t(), ids, w, gate_up, down), "unit-stride"),
        (lambda: ttn.expert_mlp(torch.randn(4, 36, device=device).half()[:, 4:], ids, w, gate_up, down), "aligned"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up, down, workspace=torch.empty(16, dtype=torch.uint8, device=device)), "workspace"),
        (lambda: ttn.expert_mlp(x, ids, w, gate_up, down, out=torch.empty(4, 32, device=device)), "out"),
    ]
    plain = torch.randn(4, 50, device=device)
    tokens = torch.zeros(4, dtype=torch.int64, device=device)
    bad += [
        (lambda: ttn.token_logprobs(plain, tokens.int()), "tokens"),
        (lambda: ttn.token_logprobs(plain, tokens[:3]), "tokens"),
        (lambda: ttn.token_logprobs(plain, tokens, top=33), "top"),
        (lambda: ttn.token_logprobs(plain, tokens, top=51), "top"),
        (lambda: ttn.token_logprobs(plain, tokens, top=-1), "top"),
        (lambda: ttn.token_logprobs(plain, tokens, scale=0.0), "scale"),
        (lambda: ttn.token_logprobs(plain, tokens, scale=math.inf), "scale"),
        (lambda: ttn.token_logprobs(torch.randn(50, 4, device=device).t(), tokens), "stride"),
        (lambda: ttn.token_logprobs(torch.empty(1, (1 << 20) + 1, device=device), tokens[:1]), "2\\^20"),
    ]
    for n, (call, message) in enumerate(bad):
        with pytest.raises(RuntimeError, match=message):
            call()
            pytest.fail(f"refusal {n} ({message}) did not raise")
