"""CPU: expert_mlp's workspace size as a caller plans with it, and refusals before any work."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("hidden,inner,experts,top_k", [(128, 512, 8, 2), (8, 1024, 64, 1), (64, 32, 8, 2), (256, 128, 8, 8),
                                                        (2048, 1024, 64, 8), (16, 4096, 1024, 32), (1032, 688, 10, 2),
                                                        (8, 1 << 14, 1, 3), (2048, 1 << 14, 64, 5)])
def test_a_workspace_for_the_largest_batch_holds_every_smaller_one(hidden, inner, experts, top_k):
    """The kernels change with the number of pairs; the bytes never fall as tokens grow."""
    from thintnpu_b200 import _lib
    size = _lib.lib().ttn_expert_mlp_workspace_size
    last = 0
    for tokens in [*range(0, 700), 1000, 4096, 100000]:
        need = size(tokens, hidden, inner, experts, top_k)
        assert need >= last and need % 256 == 0, tokens
        last = need


def test_sizes_beyond_the_kernels_are_refused_before_any_work():
    """Fake aligned addresses, never dereferenced: the call has to end in its checks (status 2),
    not in its first launch or in the look-up of a driver function (status 3 without a GPU)."""
    from thintnpu_b200 import _lib
    lib = _lib.lib()

    def mlp(tokens, hidden, top_k=1, inner=16, experts=8):
        return lib.ttn_expert_mlp(2, 1 << 20, hidden, tokens, hidden, 2 << 20, 3 << 20, top_k, 4 << 20, 5 << 20, experts,
                                  inner, 6 << 20, hidden, 7 << 20, 1 << 60, None)

    assert mlp(1 << 22, 1 << 13) == 2 and b"2^34" in lib.ttn_last_error()
    assert mlp(1 << 22, 4104) == 2 and mlp(1 << 14, 1 << 20, 2) == 2
