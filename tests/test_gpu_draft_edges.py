"""Calls of tree attention at the edges of what is documented."""

import pytest
import torch

from ajllm_amd import attention

pytestmark = pytest.mark.gpu


def test_masks_of_one_word_lie_anywhere(cuda):
    """One word a token has no step to the next: any stride."""
    gen = torch.Generator().manual_seed(1)
    q, keys, values = (torch.randn(s, generator=gen).to(cuda) for s in ((2, 4, 7, 64), (2, 2, 30, 64), (2, 2, 30, 64)))
    rows, masks = torch.tensor([20, 3], device=cuda), attention.tree_masks(torch.tensor([-1, 0, 0, 1, 2, 2, 5]))[0].to(cuda)
    want = attention.tree_attention(q, keys, values, rows, masks)
    apart = torch.zeros((7, 5), dtype=torch.int32, device=cuda)
    apart[:, 0] = masks[:, 0]
    across = torch.empty((1, 7), dtype=torch.int32, device=cuda).t().copy_(masks)
    for same in (across, apart[:, ::2][:, :1], across[None].expand(2, -1, -1)):
        assert same.stride(-1) != 1
        assert torch.equal(attention.tree_attention(q, keys, values, rows, same), want)


def test_more_key_heads_than_are_counted_are_refused(cuda):
    """2^32 + 1 key heads (all the same one) are not one."""
    q, cache = torch.zeros(1, 1, 1, 64, device=cuda), torch.zeros(1, 1, 8, 64, device=cuda).expand(1, 2 ** 32 + 1, 8, 64)
    with pytest.raises(ValueError, match="below 2\\^31"):
        attention.tree_attention(q, cache, cache, torch.zeros(1, dtype=torch.long, device=cuda), torch.ones((1, 1), dtype=torch.int32, device=cuda))
