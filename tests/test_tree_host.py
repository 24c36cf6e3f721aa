"""CPU checks of what the draft-tree operators decide on the host."""
import pytest
import torch

from torchplusplus_b200 import _native as N


@pytest.mark.parametrize("T,max_ctx", [(1, 8191), (64, 8191), (256, 0), (5, 1 << 24)])
def test_a_window_past_every_row_plans_as_none(T, max_ctx):
    """The workspace of the call is the one that the call without a window takes:
    from max_ctx + T on a window hides nothing."""
    size = lambda w: N.lib().tpp_attention_tree_workspace(1, T, 16, 8, max_ctx, 128, w)
    for w in (max_ctx + T, 2 ** 31, 2 ** 62, 2 ** 63 - 64, 2 ** 63 - 2, 2 ** 63 - 1):
        assert size(w) == size(-1)
