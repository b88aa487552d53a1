"""The token-mixing layer's parameters, without a GPU."""
import pytest
import torch

DECAYS = [4095.0, 2051.0, 511.0, 3.3]                 # none of them a bfloat16 number


@pytest.mark.parametrize('train_decay', [False, True])
@pytest.mark.parametrize('change', [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: torch.nn.Sequential(m).to(torch.bfloat16)[0],
                                    lambda m: m.to('cpu', torch.bfloat16)])
def test_decays_and_norm_stay_float32(change, train_decay):
    import lava_dl_amd.slayer as slayer
    block = slayer.block.LeakyAttention(32, 4, 16, decay=DECAYS, train_decay=train_decay, dropout=0.1)
    with torch.no_grad():
        block.norm.weight.copy_(1 + torch.arange(64) / 1000)
    weight, project = block.norm.weight.detach().clone(), block.project.weight.detach().clone()
    parameters = dict(block.named_parameters())
    block = change(block)
    assert block.decay.dtype == block.norm.weight.dtype == block.norm.bias.dtype == torch.float32
    assert torch.equal(block.decay.detach(), torch.tensor(DECAYS)) and torch.equal(block.norm.weight.detach(), weight)
    assert block.project.weight.dtype == block.back.weight.dtype == torch.bfloat16
    assert torch.equal(block.project.weight.detach(), project.bfloat16())
    assert block.initial_state(2).dtype == torch.float32
    for name, p in block.named_parameters():            # an optimizer made before goes on with the same parameters
        assert p is parameters[name]
    assert isinstance(block.decay, torch.nn.Parameter) == train_decay


def test_other_changes_reach_all_of_it():
    import lava_dl_amd.slayer as slayer
    block = slayer.block.LeakyAttention(32, 4, 16, train_decay=True).to('meta')
    assert all(p.is_meta for p in block.parameters())
    block = block.to_empty(device='cpu')
    assert not any(p.is_meta for p in block.parameters())
    block = slayer.block.LeakyAttention(32, 4, 16).to(torch.float64).float()
    assert all(p.dtype == torch.float32 for p in block.parameters()) and block.decay.dtype == torch.float32
    both = slayer.block.LeakyAttention(32, 4, 16).to('meta', torch.bfloat16)
    assert both.decay.is_meta and both.decay.dtype == torch.float32 and both.back.weight.dtype == torch.bfloat16


@pytest.mark.parametrize('decay', [[1.0, -0.5], [4096.5, 1.0], [float('nan'), 1.0]])
def test_decays_out_of_range_are_refused(decay):
    import lava_dl_amd.slayer as slayer
    with pytest.raises(ValueError, match='between 0 and 4096'):
        slayer.block.LeakyAttention(16, 2, 16, decay=decay)
    slayer.block.LeakyAttention(16, 2, 16, decay=[0.0, 4096.0])
