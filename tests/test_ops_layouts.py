"""boa_b200.ops on inputs that share memory with a state, and on strided ones."""
import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _ops():
    from boa_b200 import ops
    return ops


def test_step_inputs_inside_the_state():
    """Inputs that are parts of the state's memory are taken as they were before the step."""
    n, e = 300, 512
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    A, D = -torch.rand(e, 16, generator=g, device="cuda"), r(e)
    start = r(n, e, 16)

    def scan(state, copy):
        flat = state.view(n, -1)
        a = [flat[:, :e], flat[:, 700:700 + e], state[:, e - 1], state[:, 0], flat[:, 64:64 + e]]
        x, dt, B, C, z = (t.clone() for t in a) if copy else a
        return _ops().ssm_step(x, dt, state, A, B, C, D, z), state

    one, two = scan(start.clone(), False), scan(start.clone(), True)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])

    w, window = r(e, 4), r(n, 3, e)
    for cut in (slice(1, e + 1), slice(0, e), slice(2 * e, 3 * e)):
        s, t = window.clone(), window.clone()
        y = _ops().causal_conv_step(s.view(n, -1)[:, cut], s, w)
        z = _ops().causal_conv_step(t.view(n, -1)[:, cut].clone(), t, w)
        assert torch.equal(y, z) and torch.equal(s, t)


# ------------------------------------------------------------------- strided rows
def _slice(g, kind, nb, length, width, before, behind):
    """[nb, length, width] of random values inside wider and longer rows of NaN, on the GPU, with the strides it says."""
    ts, rows = before + width + behind, length + 3
    store = torch.full((nb, rows, ts), float("nan"), dtype=kind, device="cuda")
    t = store[:, 1:1 + length, before:before + width]
    t.copy_(torch.randn(nb, length, width, generator=g))
    assert t.stride() == (rows * ts, ts, 1)
    return t


# rank: columns in front of B and C, whose rows are rank + 32 wide; edge: columns around x, dt, z and dy
@pytest.mark.parametrize("nb,length,e,rank,edge", [(2, 37, 64, 4, 64), (2, 37, 64, 5, 64), (1, 130, 40, 4, 8), (3, 9, 64, 4, 3),
                                                  (2, 21, 33, 4, 4), (1, 300, 576, 20, 576)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_scan_of_strided_rows(nb, length, e, rank, edge, kind):
    """Outputs and all gradients, with the strides of the model's own projections (vector accesses) and with odd ones."""
    import test_ops_gpu as base
    g = torch.Generator().manual_seed(1000 * length + e + rank)
    c = base._scan_case(nb, length, e, kind, 7)
    x, dt, z, dy = (_slice(g, kind, nb, length, e, *at) for at in ((0, edge), (edge, 0), (edge, 0), (0, edge)))
    rows = torch.randn(nb, length, rank + 32, generator=g).to(kind).cuda()
    B, C = rows[..., rank:rank + 16], rows[..., rank + 16:]
    assert B.stride(1) == C.stride(1) == rank + 32
    lens = torch.tensor([length, length // 2, 0][:nb], dtype=torch.int32)
    c.update({k: v.cpu() for k, v in zip(("x", "dt", "z", "dy", "B", "C"), (x, dt, z, dy, B, C))})
    names = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")
    d = {k: c[k].cuda() for k in names}
    d.update(x=x, dt=dt, z=z, B=B, C=C)
    d = {k: v.detach().requires_grad_() for k, v in d.items()}
    assert all(d[k].stride() == t.stride() for k, t in (("x", x), ("dt", dt), ("z", z), ("B", B), ("C", C)))
    y, out = _ops().ssm_scan(*(d[k] for k in names[:8]), state=d["state"], lens=lens.cuda(), return_state=True)
    grads = torch.autograd.grad((y, out), [d[k] for k in names], (dy, c["dout"].cuda()))
    got = {"d" + k: v for k, v in zip(names, grads)}
    got.update(y=y.detach(), state=out.detach())
    base._scan_check(c, lens, got)


@pytest.mark.parametrize("nb,length,e,edge", [(2, 37, 64, 64), (3, 130, 40, 4), (2, 21, 64, 3), (2, 50, 33, 1)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_convolution_of_strided_rows(nb, length, e, edge, kind):
    import test_ops_gpu as base
    g = torch.Generator().manual_seed(2000 * length + e)
    _, w, b, s, _, ds = base._conv_case(nb, length, e, 4, kind, 8, True)
    x, dy = _slice(g, kind, nb, length, e, 0, edge), _slice(g, kind, nb, length, e, edge, 0)
    lens = torch.tensor([length, length // 2, 0][:nb], dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (x.detach(), w.cuda(), b.cuda(), s.cuda())]
    y, out = _ops().causal_conv(*leaves[:3], state=leaves[3], lens=lens.cuda(), return_state=True)
    grads = torch.autograd.grad((y, out), leaves, (dy, ds.cuda()))
    r = ref.conv(x.double().cpu(), w.double(), b.double(), True, s.double(), lens, dy.double().cpu(), ds.double())
    total = nb * length
    # the counts of test_causal_conv
    for name, got, k in zip(("y", "state", "dx", "dw", "db", "dstate"), (y, out) + grads,
                            (64, 0, 128, 192 + total / 8, 192 + total / 8, 128)):
        ref.close(name, got, *r[name], k)


@pytest.mark.parametrize("rows,width,edge", [(40, 64, 64), (300, 256, 8), (37, 96, 3), (9, 1040, 16), (20, 33, 1)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_layer_norm_of_strided_rows(rows, width, edge, kind):
    g = torch.Generator().manual_seed(3000 * rows + width)
    x, dy = _slice(g, kind, 1, rows, width, 0, edge)[0], _slice(g, kind, 1, rows, width, edge, 0)[0]
    w, b = 1 + 0.2 * torch.randn(width, generator=g), 0.2 * torch.randn(width, generator=g)
    leaves = [t.requires_grad_() for t in (x.detach(), w.cuda(), b.cuda())]
    y = _ops().layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    vals, scales = ref.norm(x.double().cpu(), w.double(), b.double(), dy.double().cpu())
    # the counts of test_layer_norm
    n = 4 * (width / 32 + 13) + 16
    m = n + rows / 8 + 64
    for name, got, v, s, k in zip(("y", "dx", "dw", "db"), (y,) + grads, vals, scales, (n, n, m, m)):
        ref.close(name, got, v, s, k)


def test_negated_views():
    """A view that torch marks as negated (the imaginary part of a conjugate) holds the other sign in memory."""
    ops = _ops()
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    neg = lambda t: torch._neg_view(-t)  # noqa: E731
    x, w, b, dy = r(6, 32), r(32), r(32), r(6, 32)
    assert neg(x).is_neg() and torch.equal(neg(x), x)
    one = [t.detach().requires_grad_() for t in (x, w, b)]
    two = [neg(t).detach().requires_grad_() for t in (x, w, b)]
    for f in (lambda x, w, b: ops.layer_norm(x, w, b),
              lambda x, w, b: ops.causal_conv(x[None], w[:, None] * torch.ones(4, device="cuda"), b),
              lambda x, w, b: ops.ssm_scan(x[None], x[None], -torch.ones(32, 16, device="cuda"), x[None, :, :16],
                                           x[None, :, 16:], w, x[None], b)):
        y, z = f(*one), f(*two)
        assert torch.equal(y, z)
        up = dy.view(y.shape)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, one, up), torch.autograd.grad(z, two, neg(up))))
    A, h, window, k = -torch.ones(32, 16, device="cuda"), r(6, 32, 16), r(6, 3, 32), r(32, 4)
    for f in (neg, lambda t: t):
        y, end = ops.ssm_scan(x[None], x[None], f(A), f(x[None, :, :16]), f(x[None, :, 16:]), state=f(h[:1]), return_state=True)
        u, win = ops.causal_conv(x[None], f(k), state=f(window[:1]), return_state=True)
        s, t = h.clone(), window.clone()
        v = ops.ssm_step(f(x), f(x), s, f(A), f(x[:, :16]), f(x[:, 16:]))
        q = ops.causal_conv_step(f(x), t, f(k))
        now = (y, end, u, win, s, t, v, q)
        if f is neg:
            first = now
    assert all(torch.equal(p, q) for p, q in zip(first, now))
    with pytest.raises(ValueError, match="in place"):
        ops.ssm_step(x, x, neg(h), A, x[:, :16], x[:, 16:])
    with pytest.raises(ValueError, match="in place"):
        ops.causal_conv_step(x, neg(window), k)
