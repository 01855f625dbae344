"""The layer-by-layer model (forward_layers / step_layers / train_step), whose
blocks run boa_b200.ops together, against the 64-bit oracle model.

Tolerance: an fp32 result of one layer here passes sums of at most 128 + 64 +
128 + 64 + 256 products and 8 roundings for each of 24 tokens, twice for a
gradient: about 2 layers * 2 * 900 roundings of 2^-24 = 2e-4 of the sums of
absolute values.  Results are compared in the 2-norm, where signs cancel as in
the sums themselves: 1e-3 of the result's norm.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle import model_oracle as mo

pytestmark = pytest.mark.gpu

REL = 1e-3


def _model(d=64, layers=2, vocab=256, seed=0):
    from model import seeded_model
    return seeded_model(d, layers, vocab, seed, weight_format=None if d in (64, 256) else "bf16").cuda()


def _leaves(m):
    return {k: v.detach().double().cpu().requires_grad_() for k, v in m.state_dict().items()}


def _reference(sd, tokens, state=None):
    """logits [B, L, vocab] of the oracle's step, with gradients."""
    cfg = mo.config_from_state_dict(sd)
    st = mo.init_state(cfg, tokens.shape[0], torch.float64) if state is None else state
    out = []
    for t in range(tokens.shape[1]):
        h = sd["embedding.weight"][tokens[:, t]]
        new = []
        for i in range(cfg.n_layers):
            p = f"blocks.{i}."
            u = mo._ln(h, sd[p + "ln1.weight"], sd[p + "ln1.bias"])
            o, c, s = mo._mixer_step(sd, p + "mamba.", cfg, u, *st[i])
            new.append((c, s))
            v = mo._ln(o, sd[p + "ln2.weight"], sd[p + "ln2.bias"])
            f = F.gelu(v @ sd[p + "ff.0.weight"].T + sd[p + "ff.0.bias"])
            h = h + f @ sd[p + "ff.2.weight"].T + sd[p + "ff.2.bias"]
        st = new
        r = torch.relu(h @ sd["head.0.weight"].T + sd["head.0.bias"])
        out.append(r @ sd["head.2.weight"].T + sd["head.2.bias"])
    return torch.stack(out, 1), st


def _near(a, b, name=""):
    a, b = a.detach().double().cpu(), b.detach()
    err = (a - b).norm() / b.norm().clamp(min=1e-30)
    assert err <= REL, (name, err.item())


def _tokens(b, n, seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(0, 256, (b, n), generator=g)


@pytest.mark.parametrize("d,layers", [(64, 2), (48, 1), (72, 1)])
def test_forward_layers_matches_oracle(d, layers):
    """Logits and the state left behind; d_model 48 and 72 are sizes that only this path runs."""
    m = _model(d, layers)
    x = _tokens(3, 24, d)
    with torch.no_grad():
        got, state = m.forward_layers(x, return_state=True)
    want, st = _reference({k: v.detach() for k, v in _leaves(m).items()}, x)
    _near(got, want, "logits")
    for (gc, gs), (wc, ws) in zip(state, st):
        _near(gc, wc.transpose(1, 2), "window")
        _near(gs, ws, "scan state")


def test_fused_kernel_agrees():
    m = _model()
    x = _tokens(4, 32, 9).cuda()
    with torch.no_grad():
        p = torch.softmax(m.forward_layers(x), -1)
    assert (p - torch.softmax(m(x), -1)).abs().max() < 1e-4


def test_prompt_then_steps_continue():
    """A prompt with states returned, then single tokens, then another piece: one sequence."""
    m = _model(48, 2)
    x = _tokens(5, 30, 1).cuda()
    with torch.no_grad():
        whole, end = m.forward_layers(x, return_state=True)
        out, state = m.forward_layers(x[:, :11], return_state=True)
        parts = [out] + [m.step_layers(x[:, t], state)[:, None] for t in range(11, 19)]
        out, state = m.forward_layers(x[:, 19:], state, return_state=True)
        first = m.init_layers(5)
        steps = torch.stack([m.step_layers(x[:, t], first) for t in range(4)], 1)
    w = whole.double().cpu()
    _near(torch.cat(parts + [out], 1), w)
    _near(steps, w[:, :4])
    for a, b in zip(state, end):
        _near(a[0], b[0].double().cpu())
        _near(a[1], b[1].double().cpu())


def test_ragged_rows_do_not_see_their_padding():
    m = _model()
    x = _tokens(4, 20, 2).cuda()
    lens = torch.tensor([20, 1, 0, 13], device="cuda")
    with torch.no_grad():
        got, state = m.forward_layers(x, lens=lens, return_state=True)
        for i, n in enumerate(lens.tolist()):
            if n == 0:
                assert all((c[i] == 0).all() and (s[i] == 0).all() for c, s in state)
                continue
            alone, st = m.forward_layers(x[i:i + 1, :n], return_state=True)
            _near(got[i, :n], alone[0].double().cpu())
            for (c, s), (ac, as_) in zip(state, st):
                _near(c[i], ac[0].double().cpu())
                _near(s[i], as_[0].double().cpu())


@pytest.mark.parametrize("lens", [None, (24, 9, 0)])
def test_parameter_gradients_match_oracle(lens):
    from train import train_step
    m = _model(48, 2, seed=3)
    sd = _leaves(m)
    batch = _tokens(3, 25, 4)
    n = None if lens is None else torch.tensor(lens) + torch.tensor([1, 1, 0])
    loss = train_step(m, batch.cuda(), torch.optim.SGD(m.parameters(), lr=0.0), F.cross_entropy, lens=n)
    logits, _ = _reference(sd, batch[:, :-1])
    targets = batch[:, 1:].clone()
    if lens is not None:
        for i, v in enumerate(lens):
            targets[i, v:] = -100
    want = F.cross_entropy(logits.reshape(-1, 256), targets.reshape(-1))
    want.backward()
    _near(loss, want, "loss")
    for k, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), k
        _near(p.grad, sd[k].grad, k)


def test_train_step_under_autocast_and_after_it_the_codec():
    """Mixed precision runs, changes every parameter, and the fused kernel takes the trained weights."""
    from train import train_step
    m = _model(64, 1)
    before = {k: v.clone() for k, v in m.state_dict().items()}
    opt = torch.optim.AdamW(m.parameters(), lr=1e-3)
    batch = _tokens(8, 33, 5).cuda()
    with torch.autocast("cuda", torch.bfloat16):
        for _ in range(2):
            loss = train_step(m, batch, opt, F.cross_entropy)
    assert torch.isfinite(loss)
    assert all(not torch.equal(before[k], v) for k, v in m.state_dict().items())
    with torch.no_grad():
        p = torch.softmax(m.forward_layers(batch), -1)
    assert (p - torch.softmax(m(batch), -1)).abs().max() < 1e-4


def test_refusals():
    from model import seeded_model
    m = seeded_model(64, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        m.forward_layers(torch.zeros(1, 4, dtype=torch.long))
    m = m.cuda()
    with pytest.raises(ValueError, match="batch, length"):
        m.forward_layers(torch.zeros(4, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError, match="batch"):
        m.step_layers(torch.zeros(1, 4, dtype=torch.long, device="cuda"), m.init_layers(1))
