"""What the token-mixing layer promises beside its formulas."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'


def test_bfloat16_is_that_of_the_projections():
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(1)
    block = slayer.block.LeakyAttention(64, 4, 16, decay=[4095.0, 2051.0, 511.0, 3.3]).to(DEV)
    by_hand = copy.deepcopy(block)
    by_hand.project.bfloat16(), by_hand.back.bfloat16()
    block = block.to(torch.bfloat16)
    x = torch.randn(3, 70, 64, device=DEV).bfloat16()
    y, state = block(x, return_state=True)
    ref, last = by_hand(x, return_state=True)
    assert y.dtype == torch.bfloat16 and state.dtype == torch.float32
    assert torch.equal(y, ref) and torch.equal(state, last)
    assert torch.equal(block.step(x[:, 0], state), by_hand.step(x[:, 0], last)) and torch.equal(state, last)
