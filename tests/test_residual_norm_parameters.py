"""The parameters of the norms around a block, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize('change', [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.half(),
                                    lambda m: torch.nn.Sequential(m, torch.nn.Linear(8, 8)).to(torch.bfloat16)[0]])
def test_weights_stay_float32(change):
    import lava_dl_amd.slayer as slayer
    norm = slayer.neuron.norm.ResidualNorm(8, scale=0.3)                     # 0.3 is no bfloat16 number
    with torch.no_grad():
        norm.weight.add_(torch.arange(8) / 1000)
    before = {k: (p, p.detach().clone()) for k, p in norm.named_parameters()}
    norm = change(norm)
    assert set(before) == {'weight', 'inner', 'scale'}
    for k, p in norm.named_parameters():
        assert p is before[k][0] and p.dtype == torch.float32 and torch.equal(p.detach(), before[k][1])
    assert all(p.is_meta for p in norm.to('meta').parameters())
