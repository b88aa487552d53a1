"""The token-mixing layer: its operators together against the same formulas in float64, in training, in parts and token by token.

Tolerance.  The layer's operators are each held to a few hundred 2^-24 of their magnitudes in tests of their own; the projections are
float32 products over at most 96 features.  The norm divides by the spread of a head's results and so passes on relative errors:
2^-24 * 2000 of the largest magnitude, for gradients (two more products each) 2^-24 * 20000."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV, U = 'cuda:0', 2.0 ** -24


def plain(block, x, mask, lengths):
    """The layer in float64 on the host."""
    n, t, _ = x.shape
    h, d = block.heads, block.head_features
    w = [p.detach().cpu().double().requires_grad_() for p in (block.project.weight, block.norm.weight, block.norm.bias, block.back.weight,
                                                               block.decay)]
    x = x.detach().cpu().double().requires_grad_()
    q, k, v = (x @ w[0].t()).reshape(n, t, 3, h, d).unbind(2)
    S, out = torch.zeros(n, h, d, d, dtype=torch.float64), []
    for s in range(t):
        on = torch.tensor([s < length for length in lengths]).reshape(n, 1, 1, 1)
        S = torch.where(on, S * (1 - w[4] / 4096)[:, None, None] + k[:, s, :, :, None] * v[:, s, :, None, :], S)
        out.append(torch.where(on[..., 0], block.scale * torch.einsum('nhk,nhkv->nhv', q[:, s], S), 0))
    y = torch.stack(out, 1)
    y = (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, unbiased=False, keepdim=True) + 1e-5)
    z = y.reshape(n, t, h * d) * w[1] + w[2]
    z = z * torch.sigmoid(z) * mask
    return z @ w[3].t(), [x] + w


def test_training_step():
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(0)
    block = slayer.block.LeakyAttention(48, 3, 32, train_decay=True, dropout=0.25, seed=5).to(DEV)
    x = torch.randn(4, 90, 48, device=DEV, requires_grad=True)
    lengths = [90, 1, 0, 64]
    g = torch.randn(4, 90, 48, device=DEV)
    y = block(x, lengths=torch.tensor(lengths, device=DEV))
    wrt = [x, block.project.weight, block.norm.weight, block.norm.bias, block.back.weight, block.decay]
    grads = torch.autograd.grad(y, wrt, g)
    mask = slayer.neuron.counter_dropout(torch.ones(4 * 90, 96, device=DEV), 0.25, 5, 0).cpu().double().reshape(4, 90, 96)
    ref, leaves = plain(block, x, mask, lengths)
    want = torch.autograd.grad(ref, leaves, g.cpu().double())
    assert float((y.detach().cpu().double() - ref).abs().max()) <= 2000 * U * float(ref.detach().abs().max())
    for a, b in zip(grads, want):
        assert a.shape == b.shape and float((a.cpu().double() - b).abs().max()) <= 20000 * U * float(b.abs().max())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_generation_goes_on_from_a_prompt(dtype):
    """bfloat16: a token's value is rounded five times on its way, 2^-8 each, and the norm takes one division by the spread."""
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(1)
    block = slayer.block.LeakyAttention(64, 4, 16, dropout=0.5).to(DEV)
    block.project.to(dtype), block.back.to(dtype)
    block.eval()
    x = torch.randn(3, 40, 64, device=DEV).to(dtype)
    with torch.no_grad():
        whole = block(x)
        y, state = block(x[:, :30], return_state=True)
        parts = [y]
        for t in range(30, 40):
            parts.append(block.step(x[:, t], state)[:, None])
        again, last = block(x[:, 30:], state=block(x[:, :30], return_state=True)[1], return_state=True)
    tol = (2000 * U if dtype == torch.float32 else 12 * 2.0 ** -8) * float(whole.abs().max())
    assert float((torch.cat(parts, 1) - whole).abs().max()) <= tol and float((again - whole[:, 30:]).abs().max()) <= tol
    assert float((last - state).abs().max()) <= 2000 * U * float(state.abs().max())
    fresh = block.initial_state(3)
    first = block.step(x[:, 0], fresh)
    assert float((first - whole[:, 0]).abs().max()) <= tol


def test_learns():
    """A few steps of gradient descent on a task that needs the memory: the sum of the last tokens' first feature."""
    import lava_dl_amd.slayer as slayer
    torch.manual_seed(2)
    block = slayer.block.LeakyAttention(16, 2, 16, train_decay=True).to(DEV)
    optim = torch.optim.Adam(block.parameters(), lr=1e-2)
    x = torch.randn(16, 64, 16, device=DEV)
    target = torch.zeros_like(x)
    target[..., 0] = torch.stack([x[:, max(0, t - 3):t + 1, 0].sum(1) for t in range(64)], 1)
    losses = []
    for _ in range(60):
        optim.zero_grad()
        loss = (block(x) - target).square().mean()
        loss.backward()
        optim.step()
        losses.append(float(loss))
    assert losses[-1] < 0.8 * losses[0]


def test_refusals():
    import lava_dl_amd.slayer as slayer
    with pytest.raises(ValueError, match='decays'):
        slayer.block.LeakyAttention(16, 2, 16, decay=[1.0])
    with pytest.raises(RuntimeError, match='128'):
        slayer.block.LeakyAttention(16, 1, 256).to(DEV)(torch.zeros(1, 2, 16, device=DEV))
