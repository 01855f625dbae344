"""Plain 64-bit references of the block operators (boa_b200.ops), position by
position from their definitions, with hand-written gradients.

Every function also gives a ``scale`` for each output: the same sums of
products with every term's absolute value.  A sum of fp32 products, computed
in any order, is off by at most (number of roundings on the longest path) *
2^-24 * scale, which is what the tests' tolerances count.
"""
import torch

N = 16


def _silu_parts(z):
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def norm(x, w, b, dy, eps=1e-5):
    """(y, dx, dw, db) and their scales, float64; b may be None."""
    n = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    r = (((x - mean) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    xh = (x - mean) * r
    # the centred value is a difference: its error is that of |x| + |mean|, which r then scales
    xs = (x.abs() + x.abs().mean(-1, keepdim=True)) * r
    y = xh * w + (0 if b is None else b)
    ys = xs * w.abs() * (1 + xh.abs()) + (0 if b is None else b.abs())
    g, gs = dy * w, (dy * w).abs()
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    dxs = r * (gs + gs.mean(-1, keepdim=True) + (xs + xh.abs()) * (gs * (xs + xh.abs())).mean(-1, keepdim=True)) * \
        (1 + xs.amax(-1, keepdim=True))
    return (y, dx, (dy * xh).sum(0), dy.sum(0)), (ys, dxs, (dy.abs() * xs * (1 + xh.abs())).sum(0), dy.abs().sum(0))


def conv(x, w, b, silu, state, lens, dy, dout):
    """{name: (value, scale)}: y, state, dx, dw, db, dstate.  state, b, lens, dout may be None."""
    B, L, E = x.shape
    K = w.shape[1]
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    ys, dxs = torch.zeros_like(x), torch.zeros_like(x)
    head = torch.zeros(B, K - 1, E, dtype=x.dtype) if state is None else state
    out, dhead, dheads = torch.zeros_like(head), torch.zeros_like(head), torch.zeros_like(head)
    dw, dws = torch.zeros_like(w), torch.zeros_like(w)
    db, dbs = torch.zeros(E, dtype=x.dtype), torch.zeros(E, dtype=x.dtype)
    bias = torch.zeros(E, dtype=x.dtype) if b is None else b
    for i in range(B):
        n = L if lens is None else int(min(max(int(lens[i]), 0), L))
        row = torch.cat([head[i], x[i, :n]])
        p = bias + sum(w[:, k] * row[k:k + n] for k in range(K))
        ps = bias.abs() + sum((w[:, k] * row[k:k + n]).abs() for k in range(K))
        f, df = _silu_parts(p) if silu else (p, torch.ones_like(p))
        y[i, :n] = f
        ys[i, :n] = f.abs() + 1.1 * ps          # |silu'| <= 1.1
        out[i] = row[n:]
        dp = dy[i, :n] * df
        dps = dy[i, :n].abs() * (1.1 + 0.5 * ps if silu else 1.0)   # |silu''| <= 0.5
        dr, drs = torch.zeros_like(row), torch.zeros_like(row)
        if dout is not None:
            dr[n:] += dout[i]
            drs[n:] += dout[i].abs()
        for k in range(K):
            dr[k:k + n] += w[:, k] * dp
            drs[k:k + n] += w[:, k].abs() * dps
            dw[:, k] += (dp * row[k:k + n]).sum(0)
            dws[:, k] += (dps * row[k:k + n].abs()).sum(0)
        db += dp.sum(0)
        dbs += dps.sum(0)
        dx[i, :n], dxs[i, :n] = dr[K - 1:], drs[K - 1:]
        dhead[i], dheads[i] = dr[:K - 1], drs[:K - 1]
    return {"y": (y, ys), "state": (out, torch.zeros_like(out)), "dx": (dx, dxs), "dw": (dw, dws), "db": (db, dbs),
            "dstate": (dhead, dheads)}


def softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))


def scan(x, dt, A, B, C, D, z, bias, plus, state, lens, dy, dout):
    """{name: (value, scale)}: y, state, dx, ddt, dA, dB, dC, dD, dz, dbias, dstate."""
    nb, L, E = x.shape
    raw = dt + (0 if bias is None else bias)
    d = softplus(raw) if plus else raw
    dd_draw = torch.sigmoid(raw) if plus else torch.ones_like(raw)
    live = torch.ones(nb, L, dtype=torch.bool)
    if lens is not None:
        live = torch.arange(L)[None] < lens.long()[:, None]
    on = live[..., None]
    zero = lambda t: torch.where(on, t, torch.zeros_like(t))  # noqa: E731
    d, x, B, C = zero(d), zero(x), zero(B), zero(C)
    gate, dgate = _silu_parts(zero(z)) if z is not None else (torch.ones_like(x), None)
    Dv = torch.zeros(E, dtype=x.dtype) if D is None else D
    g = zero(dy) * gate
    h0 = torch.zeros(nb, E, N, dtype=x.dtype) if state is None else state
    hs, ha = [h0], [h0.abs()]
    v, va = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(L):
        a = torch.exp(d[:, t, :, None] * A)
        u = (d[:, t] * x[:, t])[..., None] * B[:, t, None]
        hs.append(a * hs[-1] + u)
        ha.append(a * ha[-1] + u.abs())
        v[:, t] = (hs[-1] * C[:, t, None]).sum(-1)
        va[:, t] = (ha[-1] * C[:, t, None].abs()).sum(-1)
    v, va = v + Dv * x, va + (Dv * x).abs()
    r = {"y": (zero(v * gate), va * gate.abs()), "state": (hs[-1], ha[-1])}
    dx, dxa = Dv * g, (Dv * g).abs()
    dd, dda = torch.zeros_like(x), torch.zeros_like(x)
    dB, dBa, dC, dCa = (torch.zeros_like(B) for _ in range(4))
    dA, dAa = torch.zeros_like(A), torch.zeros_like(A)
    e = torch.zeros_like(h0) if dout is None else dout
    ea = e.abs()
    for t in reversed(range(L)):
        a = torch.exp(d[:, t, :, None] * A)
        gt, Bt, Ct = g[:, t, :, None], B[:, t, None], C[:, t, None]
        du = (d[:, t] * x[:, t])[..., None]
        e, ea = e + gt * Ct, ea + (gt * Ct).abs()
        dC[:, t], dCa[:, t] = (gt * hs[t + 1]).sum(1), (gt.abs() * ha[t + 1]).sum(1)
        dB[:, t], dBa[:, t] = (du * e).sum(1), (du.abs() * ea).sum(1)
        s1, s1a = (e * Bt).sum(-1), (ea * Bt.abs()).sum(-1)
        e, ea = e * a, ea * a
        q, qa = e * hs[t], ea * ha[t]
        dx[:, t] += s1 * d[:, t]
        dxa[:, t] += s1a * d[:, t].abs()
        dd[:, t] = s1 * x[:, t] + (q * A).sum(-1)
        dda[:, t] = s1a * x[:, t].abs() + (qa * A.abs()).sum(-1)
        dA += (q * d[:, t, :, None]).sum(0)
        dAa += (qa * d[:, t, :, None].abs()).sum(0)
    ddt, ddta = zero(dd * dd_draw), zero(dda * dd_draw)
    r.update(dx=(dx, dxa), ddt=(ddt, ddta), dA=(dA, dAa), dB=(dB, dBa), dC=(dC, dCa),
             dD=((g * x).sum((0, 1)), (g * x).abs().sum((0, 1))),
             dbias=(ddt.sum((0, 1)), ddta.sum((0, 1))), dstate=(e, ea))
    if z is not None:
        r["dz"] = (zero(zero(dy) * v * dgate), zero(dy).abs() * va * 1.1)
    return r


def close(name, got, ref, scale, roundings):
    """|got - ref| <= half a step of got's type * |ref| + roundings * 2^-24 * scale, elementwise; the
    smallest normal number covers results that the type cannot hold."""
    info = torch.finfo(got.dtype)
    g = got.detach().double().cpu()
    assert g.shape == ref.shape, (name, g.shape, ref.shape)
    assert torch.isfinite(g).all(), f"{name}: not finite"
    fp32 = roundings * 2.0 ** -24 * scale
    # the fp32 value is off by fp32, and is then rounded once to got's type
    tol = fp32 + info.eps / 2 * (ref.abs() + fp32) + info.tiny
    off = (g - ref).abs()
    bad = off > tol
    if bad.any():
        i = (off / tol).argmax().item()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; worst {g.flatten()[i]:.9g} against "
                             f"{ref.flatten()[i]:.9g}, tolerance {tol.flatten()[i]:.3g}")
