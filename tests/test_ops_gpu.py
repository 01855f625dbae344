"""boa_b200.ops on the GPU against 64-bit references (tests/ops_reference.py).

Tolerances count roundings (see ops_reference.close).  For the scan a history
of L tokens passes at most L decays; each is a rounded exponent (d * A2, off by
3 roundings relative to an exponent whose size times the decay stays below
0.4) and an ex2 (2 units in the last place = 4 roundings), a product and a sum:
8 roundings a token both for h and for its gradient, 16 L where a result
multiplies the two, plus 64 for softplus, the gate (exp of arguments up to
10: 16 roundings each) and the sums over states.
"""
import itertools

import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _ops():
    from boa_b200 import ops
    return ops


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _cuda(t, grad=False):
    if t is None:
        return None
    t = t.cuda()
    return t.requires_grad_() if grad else t


def _64(t):
    return None if t is None else t.detach().double().cpu()


# ----------------------------------------------------------------- layer norm
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 64), (16, 64), (7, 33), (300, 256), (5, 515), (37, 1000),
                                        (3, 1024), (9, 1025), (4, 4100), (2, 8192), (2500, 8), (1300, 1536)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_layer_norm(rows, width, kind):
    g = _gen(rows * 10000 + width)
    x = (0.5 + torch.randn(rows, width, generator=g)).to(kind)
    w, b = 1 + 0.2 * torch.randn(width, generator=g), 0.2 * torch.randn(width, generator=g)
    dy = torch.randn(rows, width, generator=g).to(kind)
    xs, ws, bs = _cuda(x, True), _cuda(w, True), _cuda(b, True)
    y = _ops().layer_norm(xs, ws, bs)
    grads = torch.autograd.grad(y, (xs, ws, bs), dy.cuda())
    with torch.no_grad():
        assert torch.equal(y, _ops().layer_norm(xs, ws, bs))
    vals, scales = ref.norm(_64(x), w.double(), b.double(), _64(dy))
    # sums of `width` terms in trees of depth <= width / 32 + 13; rows / 8 terms one after the other for dw and db
    n = 4 * (width / 32 + 13) + 16
    m = n + rows / 8 + 64
    for name, got, v, s, k in zip(("y", "dx", "dw", "db"), (y,) + grads, vals, scales, (n, n, m, m)):
        ref.close(name, got, v, s, k)


def test_layer_norm_views_and_leading_axes():
    ops = _ops()
    g = _gen(5)
    wide = torch.randn(4, 9, 96, generator=g).cuda()
    w, b = torch.randn(32, generator=g).cuda(), torch.randn(32, generator=g).cuda()
    for x in (wide[..., 32:64], wide[..., 1:33], wide[..., ::3], wide.transpose(0, 1)[..., :32], wide[0, 0, :32],
              wide[:, :0, :32]):
        y = ops.layer_norm(x, w, b)
        assert y.shape == x.shape
        # rows that do not start on 16 bytes are summed in another order, so the bits may differ from a contiguous
        # copy's: both are held to the 64-bit value, with test_layer_norm's count at width 32
        flat = _64(x).reshape(-1, 32)
        vals, scales = ref.norm(flat, _64(w), _64(b), torch.zeros_like(flat))
        ref.close("y", y.reshape(-1, 32), vals[0], scales[0], 72)
        ref.close("y", ops.layer_norm(x.contiguous(), w, b).reshape(-1, 32), vals[0], scales[0], 72)
    x = wide[..., 32:64].detach().requires_grad_()
    c = wide[..., 32:64].contiguous().detach().requires_grad_()
    # dy of stride 0, as sum().backward() gives
    (gx,) = torch.autograd.grad(ops.layer_norm(x, w, b).sum(), x)
    (gc,) = torch.autograd.grad(ops.layer_norm(c, w, b).sum(), c)
    assert torch.equal(gx, gc)
    assert ops.layer_norm(x, w).shape == x.shape                 # no bias
    e = torch.zeros(0, 32, device="cuda", requires_grad=True)
    ww = w.clone().requires_grad_()
    gw = torch.autograd.grad(ops.layer_norm(e, ww, b).sum(), ww)[0]
    assert torch.equal(gw, torch.zeros_like(gw))


def test_layer_norm_constant_rows_and_large_offset():
    ops = _ops()
    w, b = torch.full((48,), 2.0).cuda(), torch.full((48,), 0.25).cuda()
    y = ops.layer_norm(torch.full((3, 48), 7.0).cuda(), w, b)
    assert torch.equal(y, torch.full_like(y, 0.25))
    # the variance is summed around the mean: an offset 2^10 times the spread costs 10 bits, not 20
    x = 1024.0 + torch.randn(8, 256, generator=_gen(1))
    vals, scales = ref.norm(x.double(), torch.ones(256).double(), None, torch.zeros(8, 256).double())
    ref.close("y", ops.layer_norm(x.cuda(), torch.ones(256).cuda()), vals[0], scales[0], 100)


# --------------------------------------------------------- causal convolution
def _conv_case(B, L, E, K, kind, seed, state):
    g = _gen(seed)
    x = torch.randn(B, L, E, generator=g).to(kind)
    w, b = 0.4 * torch.randn(E, K, generator=g), 0.2 * torch.randn(E, generator=g)
    s = torch.randn(B, K - 1, E, generator=g).to(kind) if state else None
    dy = torch.randn(B, L, E, generator=g).to(kind)
    ds = torch.randn(B, K - 1, E, generator=g).to(kind)
    return x, w, b, s, dy, ds


@pytest.mark.parametrize("B,L,E,K,lens", [
    (1, 1, 1, 4, None), (2, 2, 8, 4, None), (3, 3, 16, 3, (0, 3, 1)), (2, 17, 33, 2, (5, 17)), (1, 257, 128, 4, None),
    (4, 61, 40, 4, (61, 0, 2, 60)), (2, 130, 96, 4, (-3, 1000)), (1, 5, 1030, 4, None), (70, 9, 24, 4, None),
    (3, 125, 8, 4, (125, 63, 62))])
@pytest.mark.parametrize("kind,silu,state", [(F32, True, True), (F32, False, False), (BF16, True, True),
                                             (F16, True, False)])
def test_causal_conv(B, L, E, K, lens, kind, silu, state):
    x, w, b, s, dy, ds = _conv_case(B, L, E, K, kind, B * 1000 + L, state)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    if n is not None:                       # nothing behind a row's end may be read
        for i, v in enumerate(lens):
            x[i, max(v, 0):] = float("nan")
            dy[i, max(v, 0):] = float("inf")
    xs, ws, bs, ss = _cuda(x, True), _cuda(w, True), _cuda(b, True), _cuda(s, state)
    y, out = _ops().causal_conv(xs, ws, bs, silu=silu, state=ss, lens=_cuda(n), return_state=True)
    inputs = [xs, ws, bs] + ([ss] if state else [])
    grads = torch.autograd.grad((y, out), inputs, (dy.cuda(), ds.cuda()))
    r = ref.conv(_64(x), w.double(), b.double(), silu, _64(s), n, _64(dy), _64(ds))
    total = B * L
    # p: K + 1 roundings; the gate 40 (exp of |p| <= 10); dx K more; dw, db: sums over batch and length
    for name, got, k in zip(("y", "state", "dx", "dw", "db", "dstate"), (y, out) + tuple(grads),
                            (64, 0, 128, 192 + total / 8, 192 + total / 8, 128)):
        ref.close(name, got, *r[name], k)
    with torch.no_grad():
        assert torch.equal(y, _ops().causal_conv(xs, ws, bs, silu=silu, state=ss, lens=_cuda(n)))


def test_causal_conv_continues_over_pieces():
    """Pieces with the state carried give the bits of one call."""
    x, w, b, s, _, _ = _conv_case(2, 50, 24, 4, F32, 3, True)
    x, w, b, s = x.cuda(), w.cuda(), b.cuda(), s.cuda()
    whole, end = _ops().causal_conv(x, w, b, state=s, return_state=True)
    got = []
    for t0, t1 in ((0, 1), (1, 3), (3, 3), (3, 29), (29, 50)):
        y, s = _ops().causal_conv(x[:, t0:t1], w, b, state=s, return_state=True)
        got.append(y)
    assert torch.equal(torch.cat(got, 1), whole) and torch.equal(s, end)


@pytest.mark.parametrize("B,E,K,kind,silu", [(1, 1, 4, F32, True), (16, 128, 4, F32, True), (33, 515, 3, BF16, True),
                                             (7, 64, 2, F16, False), (1000, 512, 4, BF16, True),
                                             # so many that a thread takes several streams
                                             (2401, 512, 4, BF16, True), (613, 515, 4, F32, True)])
def test_causal_conv_step(B, E, K, kind, silu):
    x, w, b, s, _, _ = _conv_case(B, 5, E, K, kind, E, True)
    wide = torch.empty(B, 5, 2 * E, dtype=kind).normal_().cuda()
    wide[..., :E] = x.cuda()
    st = s.cuda()
    got = torch.stack([_ops().causal_conv_step(wide[:, t, :E], st, w.cuda().view(E, 1, K), b.cuda(), silu=silu)
                       for t in range(5)], 1)
    whole, end = _ops().causal_conv(x.cuda(), w.cuda(), b.cuda(), silu=silu, state=s.cuda(), return_state=True)
    r = ref.conv(_64(x), w.double(), b.double(), silu, _64(s), None, torch.zeros(B, 5, E).double(), None)
    ref.close("y", got, *r["y"], 64)
    assert torch.equal(st, end)


# ----------------------------------------------------- selective state space scan
def _scan_case(B, L, E, kind, seed, gate=True, state=True):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    R = 5
    x, dt = r(B, L, E).to(kind), r(B, L, E).to(kind)
    z = r(B, L, 2 * E).to(kind)[..., E:] if gate else None
    rows = r(B, L, R + 32).to(kind)
    A = -torch.exp(torch.log(torch.arange(1, 17).float()) + 0.1 * r(E, 16))
    return dict(x=x, dt=dt, A=A, B=rows[..., R:R + 16], C=rows[..., R + 16:], D=1 + 0.1 * r(E), z=z,
                bias=-2.0 + 0.5 * r(E), state=0.3 * r(B, E, 16) if state else None,
                dy=r(B, L, E).to(kind), dout=0.3 * r(B, E, 16))


def _scan_grads(c, lens, plus=True, keep=("x", "dt", "A", "B", "C", "D", "z", "bias", "state")):
    d = {k: _cuda(c[k], k in keep and c[k] is not None) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")}
    y, out = _ops().ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"], softplus=plus,
                             state=d["state"], lens=_cuda(lens), return_state=True)
    names = [k for k in keep if d[k] is not None]
    grads = torch.autograd.grad((y, out), [d[k] for k in names], (c["dy"].cuda(), c["dout"].cuda()))
    got = {"d" + k: g for k, g in zip(names, grads)}
    got.update(y=y.detach(), state=out.detach())
    return got, d


def _scan_check(c, lens, got, plus=True):
    n = None if lens is None else lens
    r = ref.scan(*[_64(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")], plus, _64(c["state"]), n,
                 _64(c["dy"]), _64(c["dout"]))
    B, L, E = c["x"].shape
    h = 8 * L + 64
    count = {"y": h + 32, "state": h, "dx": h + 64, "ddt": 2 * h + 64, "dz": h + 64, "dstate": h + 32,
             "dA": 2 * h + B * L / 8 + 64, "dB": h + E / 8 + 64, "dC": h + E / 8 + 64, "dD": 64 + B * L / 8,
             "dbias": 2 * h + B * L / 8 + 64}
    for name, g in got.items():
        ref.close(name, g, *r[name], count[name])


@pytest.mark.parametrize("B,L,E,lens", [
    (1, 1, 1, None), (2, 1, 33, (0, 1)), (1, 7, 32, None), (2, 8, 31, (8, 3)), (3, 17, 128, (17, 0, 16)),
    (1, 64, 40, None), (2, 130, 65, (129, 130)), (1, 300, 288, None), (2, 65, 520, (1, 64)), (5, 33, 16, (-1, 99, 32, 8, 9)),
    # rows enough that neither direction splits the length
    (1300, 9, 8, None), (300, 20, 40, (20, 0, 7) * 100)])
@pytest.mark.parametrize("kind,gate,state", [(F32, True, True), (F32, False, False), (BF16, True, True),
                                             (F16, True, False)])
def test_ssm_scan(B, L, E, lens, kind, gate, state):
    c = _scan_case(B, L, E, kind, B * 1000 + L, gate, state)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    if lens is not None:                    # nothing behind a row's end may be read
        for i, v in enumerate(lens):
            for k in ("x", "dt", "B", "C", "z", "dy"):
                if c[k] is not None:
                    c[k][i, max(v, 0):] = float("nan")
    got, _ = _scan_grads(c, n)
    if lens is not None:
        for k in ("x", "dt", "B", "C", "z", "dy"):
            if c[k] is not None:
                c[k].nan_to_num_(0.0)
    _scan_check(c, n, got)


@pytest.mark.parametrize("plus,D,bias", [(False, True, True), (True, False, False), (False, False, False)])
def test_ssm_scan_optional_inputs(plus, D, bias):
    c = _scan_case(2, 40, 24, F32, 9)
    if not plus:
        c["dt"] = 0.05 + 0.2 * c["dt"].abs()
        c["bias"] = c["bias"].abs() * 0.01
    if not D:
        c["D"] = None
    if not bias:
        c["bias"] = None
    got, _ = _scan_grads(c, None, plus)
    _scan_check(c, None, got, plus)


def test_ssm_scan_forward_only_matches_training_forward():
    c = _scan_case(2, 100, 64, BF16, 4)
    got, d = _scan_grads(c, None)
    with torch.no_grad():
        y, out = _ops().ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"], state=d["state"],
                                 return_state=True)
    assert torch.equal(y, got["y"]) and torch.equal(out, got["state"])


def test_ssm_scan_long_and_split():
    """One long sequence (split over its length) against the same in pieces with the state carried, and against
    64 bits: 3000 tokens."""
    c = _scan_case(1, 3000, 40, F32, 11)
    got, d = _scan_grads(c, None)
    _scan_check(c, None, got)
    again, _ = _scan_grads(c, None)
    for k in got:
        assert torch.equal(got[k], again[k]), k          # fixed order: the same bits
    with torch.no_grad():
        s, ys = d["state"], []
        for t0, t1 in ((0, 1), (1, 700), (700, 700), (700, 3000)):
            cut = lambda k: d[k][:, t0:t1]  # noqa: E731
            y, s = _ops().ssm_scan(cut("x"), cut("dt"), d["A"], cut("B"), cut("C"), d["D"], cut("z"), d["bias"],
                                   state=s, return_state=True)
            ys.append(y)
    r = ref.scan(*[_64(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")], True, _64(c["state"]), None,
                 _64(c["dy"]), _64(c["dout"]))
    ref.close("y", torch.cat(ys, 1), *r["y"], 8 * 3000 + 96)
    ref.close("state", s, *r["state"], 8 * 3000 + 64)


def test_ssm_scan_decays_that_vanish_or_stay():
    """d so large that every decay underflows to 0, and so small that it rounds to 1."""
    c = _scan_case(1, 40, 16, F32, 12)
    c["bias"] = torch.cat([torch.full((8,), 300.0), torch.full((8,), -30.0)])
    got, _ = _scan_grads(c, None)
    _scan_check(c, None, got)


@pytest.mark.parametrize("B,E,kind", [(1, 1, F32), (16, 128, F32), (9, 515, BF16), (40, 96, F16),
                                      # so many that a thread takes several streams; the last group is not whole
                                      (613, 515, BF16), (601, 512, F32), (1187, 256, F16)])
def test_ssm_step(B, E, kind):
    """Steps from a state against 64 bits, and the state they leave."""
    c = _scan_case(B, 6, E, kind, E)
    d = {k: _cuda(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")}
    st = d["state"].clone()
    ys = [_ops().ssm_step(d["x"][:, t], d["dt"][:, t], st, d["A"], d["B"][:, t], d["C"][:, t], d["D"], d["z"][:, t],
                          d["bias"]) for t in range(6)]
    r = ref.scan(*[_64(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")], True, _64(c["state"]), None,
                 _64(c["dy"]), None)
    ref.close("y", torch.stack(ys, 1), *r["y"], 8 * 6 + 96)
    ref.close("state", st, *r["state"], 8 * 6 + 64)


# ------------------------------------------------------------- gradients by differences
def test_gradients_against_differences():
    """Central differences of the kernels' own fp32 outputs along random directions.  The loss is a sum of about
    n = 2000 products of size 1 with fp32 outputs (off by 2^-20 each, signs at random), so a difference over 2 eps
    is off by sqrt(n) 2^-20 / eps plus a third derivative's eps^2: 1 % of gradients of size sqrt(n) at eps = 1e-2."""
    ops = _ops()
    g = _gen(21)
    eps = 1e-2

    def check(f, inputs):
        inputs = [t.cuda().requires_grad_() for t in inputs]
        outs = f(*inputs)
        ups = [torch.randn(o.shape, generator=g).cuda() for o in outs]
        grads = torch.autograd.grad(outs, inputs, ups)
        loss = lambda ts: sum((o.double() * u.double()).sum() for o, u in zip(f(*ts), ups))  # noqa: E731
        with torch.no_grad():
            for i, t in enumerate(inputs):
                v = torch.randn(t.shape, generator=g).cuda()
                v /= v.norm() / grads[i].norm().clamp(min=1e-3).sqrt().clamp(max=1.0)
                up = [s + eps * v if j == i else s for j, s in enumerate(inputs)]
                down = [s - eps * v if j == i else s for j, s in enumerate(inputs)]
                want = ((loss(up) - loss(down)) / (2 * eps)).item()
                have = (grads[i].double() * v.double()).sum().item()
                assert abs(want - have) <= 0.01 * max(1.0, (grads[i].norm() * v.norm()).item()), (i, want, have)

    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    check(lambda x, w, b: (ops.layer_norm(x, w, b),), [r(20, 96), 1 + 0.1 * r(96), r(96)])
    check(lambda x, w, b, s: ops.causal_conv(x, w, b, state=s, return_state=True),
          [r(2, 30, 32), 0.4 * r(32, 4), r(32), r(2, 3, 32)])
    c = _scan_case(2, 30, 32, F32, 22)
    check(lambda x, dt, A, B, C, D, z, b, s: ops.ssm_scan(x, dt, A, B, C, D, z, b, state=s, return_state=True),
          [c[k].contiguous() for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")])


# ------------------------------------------------------------------- layouts, streams, graphs
def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_strides_and_broadcast_inputs():
    """Slices at odd offsets, permuted and expanded inputs give the bits of contiguous ones of the same vector
    width, and an expanded input's gradient is the sum over its copies."""
    ops = _ops()
    c = _scan_case(3, 21, 34, F32, 30)
    d = {k: _cuda(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")}
    f = lambda x, dt, B, C, z: ops.ssm_scan(x, dt, d["A"], B, C, d["D"], z, d["bias"])  # noqa: E731
    plain = f(*(d[k].contiguous() for k in ("x", "dt", "B", "C", "z")))
    for shift in (0, 1, 3):
        odd = {}
        for k in ("x", "dt", "B", "C", "z"):
            t = torch.full((3, 21, d[k].shape[2] + 7), float("nan"), device="cuda")
            t[..., shift:shift + d[k].shape[2]] = d[k]
            odd[k] = t[..., shift:shift + d[k].shape[2]]
        assert torch.equal(f(*(odd[k] for k in ("x", "dt", "B", "C", "z"))), plain)
    swapped = [d[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("x", "dt", "B", "C", "z")]
    assert torch.equal(f(*swapped), plain)
    inner = [d[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("x", "dt", "B", "C", "z")]
    assert torch.equal(f(*inner), plain)
    # one row of B for the whole batch
    row = d["B"][:1].detach().requires_grad_()
    full = d["B"][:1].expand(3, -1, -1).contiguous().detach().requires_grad_()
    gr, = torch.autograd.grad(f(d["x"], d["dt"], row.expand(3, -1, -1), d["C"], d["z"]).sum(), row)
    gf, = torch.autograd.grad(f(d["x"], d["dt"], full, d["C"], d["z"]).sum(), full)
    # the sum of three fp32 values: two roundings of their absolute sum
    assert ((gr - gf.sum(0, keepdim=True)).abs() <= 2 * 2.0 ** -23 * gf.abs().sum(0, keepdim=True)).all()
    x = d["x"].contiguous()
    w = 0.3 * torch.ones(34, 4, device="cuda")
    t = torch.zeros(3, 21, 41, device="cuda")
    t[..., 3:37] = x
    assert torch.equal(ops.causal_conv(t[..., 3:37], w), ops.causal_conv(x, w))


def test_offsets_beyond_32_bits():
    """Rows 2^31 elements apart, and a result of more than 2^31 elements."""
    ops = _ops()
    store = torch.zeros(2 ** 31 + 4096, dtype=BF16, device="cuda")
    far = store.as_strided((2, 40, 24), (2 ** 31, 24, 1))
    g = _gen(80)
    near = torch.randn(2, 40, 24, generator=g).to(BF16).cuda()
    far.copy_(near)
    w = torch.randn(24, 4, generator=g).cuda()
    assert torch.equal(ops.causal_conv(far, w), ops.causal_conv(near, w))
    c = _scan_case(2, 40, 24, BF16, 81)
    d = {k: _cuda(c[k]) for k in ("dt", "A", "B", "C", "D", "z", "bias")}
    f = lambda x: ops.ssm_scan(x, d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"])  # noqa: E731
    assert torch.equal(f(far), f(near))
    del store, far
    x = torch.randn(1, 2048, device="cuda", dtype=BF16).expand(2 ** 20 + 3, 2048)
    p = torch.ones(2048, device="cuda")
    y = ops.layer_norm(x, p)
    assert torch.equal(y[-1], y[0]) and torch.equal(y[2 ** 19], y[0]) and torch.equal(y[:1], ops.layer_norm(x[:1], p))


def test_same_tensor_twice():
    """One tensor in two places: its gradient is the sum of both."""
    ops = _ops()
    c = _scan_case(1, 20, 16, F32, 31)
    d = {k: _cuda(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")}
    both = d["B"].contiguous().detach().requires_grad_()
    gb, = torch.autograd.grad(ops.ssm_scan(d["x"], d["dt"], d["A"], both, both, d["D"], d["z"], d["bias"]).sum(), both)
    p, q = (both.detach().clone().requires_grad_() for _ in range(2))
    gp, gq = torch.autograd.grad(ops.ssm_scan(d["x"], d["dt"], d["A"], p, q, d["D"], d["z"], d["bias"]).sum(), (p, q))
    assert torch.equal(gb, gp + gq)


def test_parameters_of_other_types():
    """bf16 parameters are taken in fp32 and their gradients come back in bf16."""
    ops = _ops()
    x = torch.randn(6, 64, generator=_gen(3)).cuda().bfloat16()
    w = torch.randn(64, generator=_gen(4)).cuda().bfloat16().requires_grad_()
    y = ops.layer_norm(x, w)
    assert torch.equal(y, ops.layer_norm(x, w.float()))
    (g,) = torch.autograd.grad(y.sum(), w)
    assert g.dtype == BF16


def test_other_stream_and_partial_outputs():
    ops = _ops()
    c = _scan_case(2, 50, 64, F32, 33)
    want, _ = _scan_grads(c, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = _scan_grads(c, None)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(want[k], got[k]) for k in want)
    # only the final state is used: dy is taken as zero
    c["dy"] = torch.zeros_like(c["dy"])
    zero, d = _scan_grads(c, None)
    _, out = ops.ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"], state=d["state"],
                          return_state=True)
    gx, gs = torch.autograd.grad(out, (d["x"], d["state"]), c["dout"].cuda())
    assert torch.equal(gx, zero["dx"]) and torch.equal(gs, zero["dstate"])


def test_captured_and_replayed():
    """Forward, backward and steps captured into a graph and replayed on new inputs give the eager bits; two graphs
    replayed in turn do not disturb each other."""
    ops = _ops()
    cases = [_scan_case(2, 90, 48, F32, 40 + i) for i in range(4)]
    names = ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")
    want = [_scan_grads(c, None)[0] for c in cases]

    def build(c):
        d = {k: _cuda(c[k]).contiguous().detach().requires_grad_() for k in names}
        up = (c["dy"].cuda(), c["dout"].cuda())

        def work():
            y, out = ops.ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"], state=d["state"],
                                  return_state=True)
            return (y, out) + torch.autograd.grad((y, out), [d[k] for k in names], up)

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work()
        return d, up, graph, outs

    built = [build(cases[0]), build(cases[1])]
    order = ["y", "state"] + ["d" + k for k in names]
    for i, j in itertools.product((2, 3, 0, 1), (0, 1)):
        d, up, graph, outs = built[j]
        with torch.no_grad():
            for k in names:
                d[k].copy_(cases[i][k])
            up[0].copy_(cases[i]["dy"])
            up[1].copy_(cases[i]["dout"])
        built[1 - j][2].replay()
        graph.replay()
        torch.cuda.synchronize()
        for k, o in zip(order, outs):
            assert torch.equal(o, want[i][k]), (i, j, k)


def test_empty_sequences_backward():
    """No tokens: the states' gradients pass through, the parameters' are zero.  No rows: all gradients are zero."""
    ops = _ops()
    c = _scan_case(2, 0, 24, F32, 70)
    got, _ = _scan_grads(c, None)
    assert torch.equal(got["state"], c["state"].cuda()) and torch.equal(got["dstate"], c["dout"].cuda())
    assert all((got[k] == 0).all() for k in ("dA", "dD", "dbias"))
    x, w, b, s, dy, ds = _conv_case(2, 0, 8, 4, F32, 71, True)
    xs, ws, bs, ss = _cuda(x, True), _cuda(w, True), _cuda(b, True), _cuda(s, True)
    y, out = ops.causal_conv(xs, ws, bs, state=ss, return_state=True)
    g = torch.autograd.grad((y, out), (ws, bs, ss), (dy.cuda(), ds.cuda()))
    assert torch.equal(out, s.cuda()) and (g[0] == 0).all() and (g[1] == 0).all() and torch.equal(g[2], ds.cuda())
    c = _scan_case(0, 5, 24, F32, 72)
    got, _ = _scan_grads(c, None)
    assert all((got[k] == 0).all() for k in ("dA", "dD", "dbias"))
    x, w, b, _, dy, _ = _conv_case(0, 5, 8, 4, F32, 73, False)
    ws = _cuda(w, True)
    assert (torch.autograd.grad(ops.causal_conv(_cuda(x), ws).sum(), ws)[0] == 0).all()


def test_without_bias_backward():
    """The gradients without a bias are those with a bias of zero."""
    ops = _ops()
    x, w, _, _, dy, _ = _conv_case(2, 40, 24, 4, F32, 74, False)
    zero = torch.zeros(24)
    a, b = _cuda(x, True), _cuda(w, True)
    one = torch.autograd.grad(ops.causal_conv(a, b), (a, b), dy.cuda())
    two = torch.autograd.grad(ops.causal_conv(a, b, _cuda(zero)), (a, b), dy.cuda())
    assert _equal(one, two)
    v = _cuda(1 + 0.1 * torch.randn(24, generator=_gen(5)), True)
    one = torch.autograd.grad(ops.layer_norm(a, v), (a, v), dy.cuda())
    two = torch.autograd.grad(ops.layer_norm(a, v, _cuda(zero)), (a, v), dy.cuda())
    assert _equal(one, two)


def test_library_errors_and_inference_mode():
    from boa_b200 import _native as _n
    ops = _ops()
    with pytest.raises(_n.BoaError, match="width must be at most 8192") as e:
        ops.layer_norm(torch.zeros(1, 8193, device="cuda"), torch.ones(8193, device="cuda"))
    assert e.value.code == _n.BOA_ERR_UNSUPPORTED
    with torch.inference_mode():
        st = torch.zeros(2, 3, 8, device="cuda")
        x = torch.ones(2, 8, device="cuda")
        ops.causal_conv_step(x, st, torch.ones(8, 4, device="cuda"))
    assert torch.equal(st[:, 2], x) and (st[:, :2] == 0).all()
    # its own state again from outside is refused before anything is written
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        ops.causal_conv_step(x, st, torch.ones(8, 4, device="cuda"))
    assert (st[:, :2] == 0).all()


def test_second_derivatives_are_refused():
    ops = _ops()
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, torch.ones(16, device="cuda"))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_steps_refuse_gradients_and_saved_states_notice_them():
    """The step forms change their state in place: they refuse gradients, and a graph that saved the state as it was
    refuses to go back."""
    ops = _ops()
    c = _scan_case(2, 1, 16, F32, 60)
    d = {k: _cuda(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")}
    one = lambda k: d[k][:, 0]  # noqa: E731
    step = lambda: ops.ssm_step(one("x"), one("dt"), d["state"], d["A"], one("B"), one("C"))  # noqa: E731
    d["A"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        step()
    y = ops.ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], state=d["state"])
    with torch.no_grad():
        step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_two_calls_on_two_streams():
    """The same call on two streams at once: no scratch is shared."""
    c = _scan_case(1, 2000, 64, F32, 50)
    want, _ = _scan_grads(c, None)
    d = {k: _cuda(c[k]) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "state")}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    with torch.no_grad():
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                got.append(_ops().ssm_scan(d["x"], d["dt"], d["A"], d["B"], d["C"], d["D"], d["z"], d["bias"],
                                           state=d["state"]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want["y"]) for y in got)
