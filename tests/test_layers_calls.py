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


# ------------------------------------------------------------------- autocast
class _Small(torch.nn.Module):
    """A predictor with forward_layers that runs anywhere."""

    def __init__(self):
        super().__init__()
        self.embedding = torch.nn.Embedding(256, 16)
        self.head = torch.nn.Linear(16, 256)

    def forward_layers(self, x, lens=None):
        return self.head(self.embedding(x.long()))


def _steps(m, batches, dev, around_all):
    """One optimizer step a batch in bf16: all in one autocast region, or each in its own."""
    from train import train_step
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    losses = []
    if around_all:
        with torch.autocast(dev, torch.bfloat16):
            for b in batches:
                losses.append(train_step(m, b, opt, F.cross_entropy))
            last = m.forward_layers(batches[0].to(dev))         # sees the weights of the last step
    else:
        for b in batches:
            with torch.autocast(dev, torch.bfloat16):
                losses.append(train_step(m, b, opt, F.cross_entropy))
        with torch.autocast(dev, torch.bfloat16):
            last = m.forward_layers(batches[0].to(dev))
    return losses, last.detach(), {k: v.detach().clone() for k, v in m.state_dict().items()}


def _same_steps(make, dev, tolerance):
    batches = [_bytes(4, 12, 20 + i) for i in range(3)]
    one, two = (_steps(make(), batches, dev, around) for around in (True, False))
    for a, b in zip(one[0] + [one[1]] + list(one[2].values()), two[0] + [two[1]] + list(two[2].values())):
        assert (a - b).float().norm() <= tolerance * b.float().norm()


def test_steps_in_one_autocast_region_use_their_own_weights():
    """Autocast keeps the bf16 copies of weights for as long as the region lasts; a step changes the weights."""
    def make():
        torch.manual_seed(0)
        return _Small()
    _same_steps(make, "cpu", 0.0)


@pytest.mark.gpu
def test_steps_in_one_autocast_region_use_their_own_weights_gpu():
    """With forward_layers.  The embedding's gradient is summed by torch in no fixed order; a weight that moves by one
    fp32 rounding can move its bf16 copy by one step of 2^-8, few of them do."""
    _same_steps(lambda: _model(64, 1).cuda(), "cuda", 1e-3)


def test_backward_and_optimizer_run_outside_autocast():
    m = _Small()
    seen = []
    m.head.weight.register_hook(lambda g: seen.append(torch.is_autocast_enabled("cpu")))
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    opt.register_step_pre_hook(lambda *a: seen.append(torch.is_autocast_enabled("cpu")))
    from train import train_step
    with torch.autocast("cpu", torch.bfloat16):
        train_step(m, _bytes(2, 5, 3), opt, F.cross_entropy)
        assert torch.is_autocast_enabled("cpu")
    assert seen == [False, False]


# ------------------------------------------------------------------- captured steps
def _capture_step(m, batch):
    """A graph of one optimizer step, behind the steps on another stream that such a capture wants."""
    from train import train_step
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    step = lambda: train_step(m, batch, opt, F.cross_entropy)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    return graph, loss


@pytest.mark.gpu
def test_fused_kernel_takes_the_weights_of_replayed_steps():
    """A replay changes the parameters without moving their versions; the fused kernel's copy of them follows."""
    m = _model(64, 1).cuda()
    batch = _bytes(4, 17, 30).cuda()
    graph, loss = _capture_step(m, batch)

    def agree():
        with torch.no_grad():
            p = torch.softmax(m.forward_layers(batch), -1)
        assert (p - torch.softmax(m(batch), -1)).abs().max() < 1e-4
        return p

    before, losses = agree(), []
    for _ in range(3):
        graph.replay()
        losses.append(loss.clone())
        after = agree()
        assert (after - before).abs().max() > 1e-3          # the step did change the model
        before = after
    assert torch.isfinite(torch.stack(losses)).all()
    handle = m.native()
    assert m.native() is handle                             # and is made once for the same weights


@pytest.mark.gpu
def test_a_step_is_not_captured_over_a_living_graph():
    """An output of an earlier call keeps its graph, whose gradients are added on the default stream: refused before
    anything is captured.  Without it the step is captured."""
    from boa_b200 import ops
    from train import train_step
    m = _model(64, 1).cuda()
    batch = _bytes(2, 9, 31).cuda()
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    assert not ops.held_on_default_stream(m.parameters())
    kept = m.forward_layers(batch)
    assert ops.held_on_default_stream(m.parameters())
    before = [p.detach().clone() for p in m.parameters()]
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            train_step(m, batch, opt, F.cross_entropy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(m.parameters(), before))
    train_step(m, batch, opt, F.cross_entropy)              # outside of a capture nothing is refused
    del kept
    assert not ops.held_on_default_stream(m.parameters())
    graph, loss = _capture_step(m, batch)
    graph.replay()
    assert torch.isfinite(loss)


# ------------------------------------------------------------------- states of another model
def test_states_of_another_depth_are_refused():
    """One state a block: fewer left the last blocks out of a step, more were ignored."""
    m = _model(64, 2)
    one = m.init_layers(3)
    for bad in (one[:1], one + one[:1], []):
        with pytest.raises(ValueError, match="2 blocks"):
            m._check_state("step_layers", bad)
    m._check_state("step_layers", one)


@pytest.mark.gpu
def test_states_of_another_depth_are_refused_gpu():
    m = _model(64, 2).cuda()
    x = _bytes(3, 4, 40).cuda()
    state = m.init_layers(3)
    for bad in (state[:1], state + state[:1]):
        with pytest.raises(ValueError, match="2 blocks"):
            m.step_layers(x[:, 0], bad)
        with pytest.raises(ValueError, match="2 blocks"):
            m.forward_layers(x, bad)
    assert all(not t.any() for s in state for t in s)
    with torch.no_grad():
        m.forward_layers(x, state)
        m.step_layers(x[:, 0], state)


# ------------------------------------------------------------------- gradients with vector accesses throughout
@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [None, (20, 7, 0)])
def test_parameter_gradients_match_oracle_at_aligned_sizes(d, lens):
    """d_model 64 and 128, whose projections' rows the scan reads and whose gradients it writes by vectors."""
    import test_layers_gpu as base
    from train import train_step
    m = base._model(d, 1, seed=5) if d == 64 else _model128()
    sd = base._leaves(m)
    batch = _bytes(3, 21, 50)
    n = None if lens is None else torch.tensor(lens) + torch.tensor([1, 1, 0])
    loss = train_step(m, batch.cuda(), torch.optim.SGD(m.parameters(), lr=0.0), F.cross_entropy, lens=n)
    logits, _ = base._reference(sd, batch[:, :-1])
    targets = batch[:, 1:].clone()
    if lens is not None:
        for i, v in enumerate(lens):
            targets[i, v:] = -100
    want = F.cross_entropy(logits.reshape(-1, 256), targets.reshape(-1))
    want.backward()
    base._near(loss, want, "loss")
    for k, p in m.named_parameters():
        base._near(p.grad, sd[k].grad, k)


def _model128():
    from model import seeded_model
    return seeded_model(128, 1, 256, 5, weight_format="bf16").cuda()


# ------------------------------------------------------------------- steps under autocast
def test_first_state_has_the_type_of_the_region():
    m = _model(64, 1)
    kinds = lambda s: [t.dtype for t in s[0]]  # noqa: E731
    with torch.autocast("cpu", torch.bfloat16):
        assert kinds(m.init_layers(2)) == [torch.bfloat16, torch.float32]
        assert kinds(m.init_layers(2, torch.float16)) == [torch.float16, torch.float32]
    assert kinds(m.init_layers(2)) == [torch.float32, torch.float32]


@pytest.mark.gpu
def test_steps_under_autocast():
    """Single tokens from the first state, in bf16, against the prompt: one sequence.  A layer's 2^-9 roundings of
    bf16 values differ where fp32 values lie on the other side of one: about 10 of them a logit, in the 2-norm."""
    m = _model(64, 1).cuda()
    x = _bytes(3, 12, 60).cuda()
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        whole = m.forward_layers(x).float()
        state = m.init_layers(3)
        steps = torch.stack([m.step_layers(x[:, t], state) for t in range(12)], 1).float()
    assert (whole - steps).norm() <= 10 * 2.0 ** -9 * whole.norm()
