"""Calls of the layer-by-layer model that its documentation allows: padding of
any value, steps under autocast, captured steps, states of another model."""
import pytest
import torch
import torch.nn.functional as F


def _model(d=64, layers=2, seed=0):
    from model import seeded_model
    return seeded_model(d, layers, 256, seed)


def _bytes(b, n, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(0, 256, (b, n), generator=g)


# ------------------------------------------------------------------- padding
def _padded():
    """Rows of 7, 0 and 4 tokens, with values behind them that no embedding has, and the same with zeros there."""
    lens = torch.tensor([7, 0, 4])
    x = _bytes(3, 7, 1)
    live = torch.arange(7) < lens[:, None]
    return x.masked_fill(~live, 0), torch.where(live, x, torch.tensor([[-100], [2 ** 40], [256]])), lens


def test_padding_is_not_embedded():
    m = _model(64, 1)
    zeros, other, lens = _padded()
    with torch.no_grad():
        assert torch.equal(m._embed(other, lens), m._embed(zeros, lens))
        assert torch.equal(m._embed(zeros), m.embedding(zeros))
    with pytest.raises(ValueError, match="lens must have shape"):
        m._embed(zeros, lens[:2])


@pytest.mark.gpu
def test_padding_takes_no_part():
    """Logits in front of each row's end, states, loss and gradients do not depend on the padding's value."""
    from train import train_step
    zeros, other, lens = _padded()
    out = []
    for x in (zeros, other):
        m = _model(64, 1).cuda()
        with torch.no_grad():
            y, s = m.forward_layers(x.cuda(), lens=lens.cuda(), return_state=True)
        loss = train_step(m, x, torch.optim.SGD(m.parameters(), lr=0.1), F.cross_entropy, lens=lens)
        out.append([y[0], y[2, :4], s[0][0], s[0][1], loss] + [p.grad for p in m.parameters()])
    # the embedding's gradient is summed by torch in no fixed order: some rounding of its largest values
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and (a - b).norm() <= 1e-6 * b.norm()
