"""GPU: the language-model operators where magnitudes are far apart or far from one, against
their 64-bit restatements (oracle/lm.py), with the tolerances of test_lm_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

from test_lm_gpu import check_route

pytestmark = pytest.mark.gpu

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
