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


def test_tree_mask_of_a_window():
    from torchplusplus_b200.llmops import tree_mask
    #      0
    #    1   2
    #   3    4 5
    #   6
    par = torch.tensor([-1, 0, 0, 1, 2, 2, 3])
    mask, depth = tree_mask(par, window_left=1)
    assert depth.tolist() == [0, 1, 1, 2, 2, 2, 3] == tree_mask(par)[1].tolist()
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1010, 0b10100, 0b100100, 0b1001000]
    assert tree_mask(par, window_left=0)[0][:, 0].tolist() == [1 << i for i in range(7)]
    for w in (-1, 3, 2 ** 40):
        assert torch.equal(tree_mask(par, window_left=w)[0], tree_mask(par)[0])
    chain = torch.arange(-1, 199).expand(2, 200)
    mask, depth = tree_mask(chain, 70)
    j = torch.arange(200)
    see = (mask[..., j // 64] >> (j % 64)) & 1
    assert torch.equal(see[1].bool(), (j <= j[:, None]) & (j >= j[:, None] - 70))
