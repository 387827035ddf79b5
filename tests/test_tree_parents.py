"""Parents of drafted tokens that are none are refused on the host."""

import pytest
import torch


@pytest.mark.parametrize("parents", [[0], [1, -1], [-1, 5], [-1, 1], [-3], [-1, -9], [-2, 0], [-1, -2, 1], [-1, 0, 3, 0]])
def test_parents_that_are_not_below_are_refused(parents):
    from turbopress_amd import tree_ancestors
    for given in (parents, [[-1] * len(parents), parents], [[parents]]):
        with pytest.raises(ValueError, match="parents of token"):
            tree_ancestors(torch.tensor(given))


def test_parents_of_no_tokens_and_of_63():
    from turbopress_amd import tree_ancestors
    assert tree_ancestors(torch.full((3, 64), -2)).tolist() == [[0] * 64] * 3
    assert tree_ancestors(torch.tensor([-1] * 63 + [62])).tolist()[63] == (1 << 62) - (1 << 63)
    assert tree_ancestors(torch.tensor([-1] * 64)).tolist() == [*(1 << i for i in range(63)), -1 << 63]
    # (63 drafted tokens behind the last: the sign's bit is a token)
    chain = torch.arange(64) - 1
    assert tree_ancestors(chain)[63] == -1
    with pytest.raises(ValueError, match="token 63"):
        tree_ancestors(torch.cat((chain[:63], torch.tensor([63]))))


@pytest.mark.gpu
def test_parents_on_the_device_are_as_documented(cuda):
    from turbopress_amd import tree_ancestors
    parents = torch.tensor([[5, 1, 9, -9, 3, -2]], device=cuda)
    assert tree_ancestors(parents).tolist() == [[1, 3, 7, 0, 16, 0]]
    assert tree_ancestors(parents[:0]).shape == (0, 6)
