"""GPU: the language-model operators where magnitudes are far apart or far from one, against
their 64-bit restatements (oracle/lm.py), with the tolerances of test_lm_gpu.py."""
from __future__ import annotations

import math

import pytest
import torch

from test_lm_gpu import check_route

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------ route_experts

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
