"""The operators of a Mamba block outside its matrix products, as measured cases:

* ``norm``       layer norm over the last axis (ln1 / ln2 of a block),
* ``conv``       the short causal depthwise convolution with SiLU over whole sequences,
* ``conv_step``  the same for one token per stream, with its window state,
* ``scan``       the selective state space scan over whole sequences,
* ``scan_step``  the same for one token per stream, with its state.

Where ``own`` is false ``run`` computes them in elementary torch operations
(fp32, long sums in fp64); where it is true it calls ``boa_b200.ops``.
"""
import math
import os
import sys

import torch

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "boa-constrictor_b200")

own = False

_N = 16        # states per channel
_K = 4         # convolution width
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # ln1 for one byte of each of 16 chunks, d_model 64: the latency of a serving step
        {"name": "norm_step", "op": "norm", "rows": 16, "width": 64, "type": "fp32", "grad": False},
        # ln1 of a training step: 32 chunks of 4096 bytes at d_model 256
        {"name": "norm_train", "op": "norm", "rows": 32 * 4096, "width": 256, "type": "bf16", "grad": True},
        # one whole chunk of a 64 MiB file cut into 1000 (67109 bytes), d_model 256, fp32 as the default model is kept
        {"name": "conv_prompt", "op": "conv", "batch": 1, "length": 67109, "channels": 512, "type": "fp32",
         "grad": False, "ragged": False, "state": True},
        # a padded training batch: 32 chunks of up to 4096 bytes, d_model 256
        {"name": "conv_train", "op": "conv", "batch": 32, "length": 4096, "channels": 512, "type": "bf16",
         "grad": True, "ragged": True, "state": False},
        # one byte of each of 16 chunks, d_model 64
        {"name": "conv_step_few", "op": "conv_step", "batch": 16, "channels": 128, "type": "fp32"},
        # one byte of each of 8192 chunks in flight, d_model 256
        {"name": "conv_step_many", "op": "conv_step", "batch": 8192, "channels": 512, "type": "bf16"},
        # a short ragged prompt of 16 chunks, d_model 64: latency again
        {"name": "scan_short", "op": "scan", "batch": 16, "length": 17, "channels": 128, "type": "fp32",
         "grad": False, "ragged": True, "state": True},
        # the chunk of conv_prompt through the scan: one sequence only, so the work has to be split over its length
        {"name": "scan_prompt", "op": "scan", "batch": 1, "length": 67109, "channels": 512, "type": "fp32",
         "grad": False, "ragged": False, "state": True},
        # the training batch of conv_train through the scan, forward and backward
        {"name": "scan_train", "op": "scan", "batch": 32, "length": 4096, "channels": 512, "type": "bf16",
         "grad": True, "ragged": True, "state": False},
        # a few odd-length pieces of long chunks at d_model 512, state carried in and out, fp32 gradients
        {"name": "scan_train_odd", "op": "scan", "batch": 3, "length": 1021, "channels": 1024, "type": "fp32",
         "grad": True, "ragged": False, "state": True},
        # one byte of each of 16 chunks, d_model 64
        {"name": "scan_step_few", "op": "scan_step", "batch": 16, "channels": 128, "type": "fp32"},
        # one byte of each of 8192 chunks in flight, d_model 256
        {"name": "scan_step_many", "op": "scan_step", "batch": 8192, "channels": 512, "type": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan", "scan", "conv_step", "scan_step"])
    kind = rng.choice(sorted(_TYPES))
    if op == "norm":
        width = _log(rng, 1, 2048)
        return {"op": op, "rows": _log(rng, 1, min(131072, 33_000_000 // width)), "width": width, "type": kind,
                "grad": rng.random() < 0.6}
    if op in ("conv_step", "scan_step"):
        return {"op": op, "batch": _log(rng, 1, 4096), "channels": _log(rng, 16, 1024), "type": kind}
    channels, length = _log(rng, 16, 1024), _log(rng, 1, 32768)
    most = 32 * 4096 * 512 if op == "conv" else 32_000_000
    return {"op": op, "batch": _log(rng, 1, max(1, min(64, most // (channels * length)))), "length": length,
            "channels": channels, "type": kind, "grad": rng.random() < 0.5, "ragged": rng.random() < 0.5,
            "state": rng.random() < 0.5}


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    op = case["op"]
    if op == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        if case["grad"]:                  # forward x -> y, backward x, dy -> dx, dw, db
            return {"bytes": 5 * n * size + 16 * d, "flops": 20 * n}
        return {"bytes": 2 * n * size + 8 * d, "flops": 8 * n}
    b, e = case["batch"], case["channels"]
    if op == "conv_step":                 # window read and written, x -> y
        return {"bytes": b * e * size * (2 * (_K - 1) + 2) + 4 * e * (_K + 1), "flops": b * e * (2 * _K + 5)}
    if op == "scan_step":                 # state read and written, x, dt, z -> y, B, C
        return {"bytes": b * e * (8 * _N + 4 * size) + 2 * b * _N * size + 4 * e * (_N + 2),
                "flops": b * e * (7 * _N + 12)}
    n = b * case["length"] * e
    if op == "conv":
        state = 2 * b * (_K - 1) * e * size if case["state"] else 0
        if case["grad"]:
            return {"bytes": 5 * n * size + 8 * e * (_K + 1) + 2 * state, "flops": n * (6 * _K + 20)}
        return {"bytes": 2 * n * size + 4 * e * (_K + 1) + state, "flops": n * (2 * _K + 5)}
    bc = 2 * b * case["length"] * _N * size
    state = 8 * b * e * _N if case["state"] else 0
    if case["grad"]:                      # forward x, dt, z, B, C -> y; backward those and dy -> all their gradients
        return {"bytes": 11 * n * size + 3 * bc + 8 * e * (_N + 2) + 2 * state, "flops": n * (26 * _N + 40)}
    return {"bytes": 4 * n * size + bc + 4 * e * (_N + 2) + state, "flops": n * (7 * _N + 12)}


# ------------------------------------------------------------------- inputs
def _parameters(channels, gen):
    """A block's recipe for A, D and the bias of dt, moved off its initial values as training does."""
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    dt = torch.exp(torch.rand(channels, generator=gen, device="cuda") * math.log(100.0) + math.log(1e-3))
    states = torch.arange(1, _N + 1, device="cuda", dtype=torch.float32)
    return {"A": -torch.exp(torch.log(states) + 0.1 * r(channels, _N)), "D": 1.0 + 0.1 * r(channels),
            "dt_bias": dt + torch.log(-torch.expm1(-dt))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind = _TYPES[case["type"]]
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    s = {"case": case}
    op = case["op"]
    if op == "norm":
        s["x"] = (0.3 + r(case["rows"], case["width"])).to(kind)
        s["weight"], s["bias"] = 1.0 + 0.1 * r(case["width"]), 0.1 * r(case["width"])
        names = ["x", "weight", "bias"]
        if case["grad"]:
            s["dy"] = r(case["rows"], case["width"]).to(kind)
    elif op in ("conv_step", "conv"):
        b, e = case["batch"], case["channels"]
        at = (b, case["length"]) if op == "conv" else (b,)
        # x is the first half of the input projection's rows
        s["x"] = r(*at, 2 * e).to(kind)[..., :e]
        s["weight"], s["bias"] = 0.3 * r(e, _K), 0.1 * r(e)
        names = ["x", "weight", "bias"]
        if op == "conv_step" or case["state"]:
            s["state"] = r(b, _K - 1, e).to(kind)
            names.append("state")
    else:
        b, e = case["batch"], case["channels"]
        at = (b, case["length"]) if op == "scan" else (b,)
        rank = -(-e // 32)
        s["x"] = torch.nn.functional.silu(r(*at, e)).to(kind)
        s["dt"] = (0.5 * r(*at, e)).to(kind)
        s["z"] = r(*at, 2 * e).to(kind)[..., e:]            # second half of the input projection's rows
        rows = r(*at, rank + 2 * _N).to(kind)               # rows of the projection that gives dt, B and C
        s["B"], s["C"] = rows[..., rank:rank + _N], rows[..., rank + _N:]
        s.update(_parameters(e, gen))
        names = ["x", "dt", "A", "B", "C", "D", "z", "dt_bias"]
        if op == "scan_step" or case["state"]:
            s["state"] = 0.1 * r(b, e, _N)
            names.append("state")
    if case.get("ragged"):
        s["lens"] = torch.randint(case["length"] // 2, case["length"] + 1, (case["batch"],), generator=gen,
                                  device="cuda", dtype=torch.int32)
        s["lens"][0] = case["length"]
    if case.get("grad"):
        if op != "norm":
            s["dy"] = r(*s["x"].shape).to(kind)
            if case["state"]:
                s["dstate"] = 0.1 * r(*s["state"].shape).to(s["state"].dtype)
        s["names"] = names
        for n in names:
            s[n] = s[n].detach().requires_grad_()
    return s


# ---------------------------------------------------------------- this repository's operators
def _ops():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from boa_b200 import ops
    return ops


def _run_own(s):
    ops = _ops()
    op = s["case"]["op"]
    if op == "conv_step":
        return ops.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"]), s["state"]
    if op == "scan_step":
        y = ops.ssm_step(s["x"], s["dt"], s["state"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"])
        return y, s["state"]
    if op == "norm":
        out = ops.layer_norm(s["x"], s["weight"], s["bias"])
    elif op == "conv":
        out = ops.causal_conv(s["x"], s["weight"], s["bias"], state=s.get("state"), lens=s.get("lens"),
                              return_state=s["case"]["state"])
    else:
        out = ops.ssm_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"],
                           state=s.get("state"), lens=s.get("lens"), return_state=s["case"]["state"])
    out = out if isinstance(out, tuple) else (out,)
    if not s["case"]["grad"]:
        return out
    up = (s["dy"], s["dstate"]) if len(out) == 2 else (s["dy"],)
    grads = torch.autograd.grad(out, [s[n] for n in s["names"]], up)
    return tuple(o.detach() for o in out) + tuple(grads)


# ---------------------------------------------------------------- plain forms
def _norm(s):
    x, w = s["x"].float(), s["weight"]
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = (hat * w + s["bias"]).to(s["x"].dtype)
    if not s["case"]["grad"]:
        return (y,)
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    dw = (dy * hat).sum(0, dtype=torch.float64).float()
    db = dy.sum(0, dtype=torch.float64).float()
    return y, dx.to(y.dtype), dw, db


def _valid(s):
    """[batch, length, 1] truth values: the positions in front of each row's end."""
    b, length = s["x"].shape[:2]
    lens = s["lens"] if "lens" in s else torch.full((b,), length, device="cuda", dtype=torch.int32)
    return (torch.arange(length, device="cuda")[None, :] < lens[:, None])[..., None], lens.long()


def _windows(s):
    """[batch, length + K - 1, channels]: the inputs behind the earlier ones, zero past each row's end."""
    b, length, e = s["x"].shape
    valid, lens = _valid(s)
    head = s["state"].float() if "state" in s else torch.zeros(b, _K - 1, e, device="cuda")
    return torch.cat([head, torch.where(valid, s["x"].float(), 0.0)], 1), valid, lens


def _conv(s):
    x, w = s["x"], s["weight"]
    length = x.shape[1]
    full, valid, lens = _windows(s)
    taps = torch.stack([full[:, 0:length], full[:, 1:length + 1], full[:, 2:length + 2], full[:, 3:length + 3]], -1)
    p = (taps * w).sum(-1) + s["bias"]
    sig = 1.0 / (1.0 + torch.exp(-p))
    out = [torch.where(valid, p * sig, 0.0).to(x.dtype)]
    last = lens[:, None] + torch.arange(_K - 1, device="cuda")[None, :]       # rows of `full` that the final window holds
    pick = last[..., None].expand(-1, -1, x.shape[2])
    if s["case"]["state"]:
        out.append(full.gather(1, pick).to(x.dtype))
    if not s["case"]["grad"]:
        return tuple(out)
    dp = torch.where(valid, s["dy"].float() * (sig * (1.0 + p * (1.0 - sig))), 0.0)
    dfull = torch.zeros_like(full)
    if s["case"]["state"]:
        dfull.scatter_add_(1, pick, s["dstate"].float())
    dfull[:, 0:length] += dp * w[:, 0]
    dfull[:, 1:length + 1] += dp * w[:, 1]
    dfull[:, 2:length + 2] += dp * w[:, 2]
    dfull[:, 3:length + 3] += dp * w[:, 3]
    dx = torch.where(valid, dfull[:, _K - 1:], 0.0).to(x.dtype)
    dw = (dp[..., None] * taps).sum((0, 1), dtype=torch.float64).float()
    out += [dx, dw, dp.sum((0, 1), dtype=torch.float64).float()]
    if s["case"]["state"]:
        out.append(dfull[:, :_K - 1].to(s["state"].dtype))
    return tuple(out)


def _conv_step(s):
    window = torch.cat([s["state"].float(), s["x"].float()[:, None]], 1)
    p = (window * s["weight"].T).sum(1) + s["bias"]
    s["state"].copy_(window[:, 1:])
    return (p / (1.0 + torch.exp(-p))).to(s["x"].dtype), s["state"]


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def _scan_step(s):
    d = _softplus(s["dt"].float() + s["dt_bias"])
    x, z = s["x"].float(), s["z"].float()
    h = torch.exp(d[..., None] * s["A"]) * s["state"] + (d * x)[..., None] * s["B"].float()[:, None]
    s["state"].copy_(h)
    v = (h * s["C"].float()[:, None]).sum(-1) + s["D"] * x
    return (v * z / (1.0 + torch.exp(-z))).to(s["x"].dtype), s["state"]


def _recurrence(decay, value):
    """h_t = decay_t h_{t-1} + value_t along the second axis, from 0, by doubling; overwrites both."""
    span = 1
    while span < value.shape[1]:
        value[:, span:] += decay[:, span:] * value[:, :-span]
        decay[:, span:] = decay[:, span:] * decay[:, :-span]
        span *= 2
    return value


def _scan(s):
    kind, (b, length, e) = s["x"].dtype, s["x"].shape
    valid, lens = _valid(s)
    zero = lambda v: torch.where(valid, v.float(), 0.0)  # noqa: E731
    x, z, B, C = zero(s["x"]), zero(s["z"]), zero(s["B"]), zero(s["C"])
    raw = s["dt"].float() + s["dt_bias"]
    d = zero(_softplus(raw))                                  # past a row's end: decay 1, nothing added
    start = s["state"] if "state" in s else torch.zeros(b, e, _N, device="cuda")
    decay = torch.exp(d[..., None] * s["A"])
    value = (d * x)[..., None] * B[:, :, None]
    value[:, 0] += decay[:, 0] * start
    h = _recurrence(decay.clone(), value)
    v = (h * C[:, :, None]).sum(-1) + s["D"] * x
    sig = 1.0 / (1.0 + torch.exp(-z))
    out = [zero(v * z * sig).to(kind)]
    if s["case"]["state"]:
        out.append(h[:, -1].clone())
    if not s["case"]["grad"]:
        return tuple(out)
    dy = zero(s["dy"])
    g = dy * z * sig
    dz = dy * v * (sig * (1.0 + z * (1.0 - sig)))
    # e_t = g_t C_t + decay_{t+1} e_{t+1}, run backwards
    add = g[..., None] * C[:, :, None]
    if s["case"]["state"]:
        add[:, -1] += s["dstate"]
    after = torch.cat([decay[:, 1:], torch.zeros_like(decay[:, :1])], 1).flip(1)
    back = _recurrence(after, add.flip(1)).flip(1)
    del add, after
    dC = (g[..., None] * h).sum(2)
    dB = ((d * x)[..., None] * back).sum(2)
    s1 = (back * B[:, :, None]).sum(-1)
    before = torch.cat([start[:, None], h[:, :-1]], 1)
    back *= decay
    q = back * before
    dd = s1 * x + (q * s["A"]).sum(-1)
    ddt = zero(dd / (1.0 + torch.exp(-raw)))
    dx = s1 * d + s["D"] * g
    dA = (q * d[..., None]).sum((0, 1), dtype=torch.float64).float()
    dD = (g * x).sum((0, 1), dtype=torch.float64).float()
    out += [zero(dx).to(kind), ddt.to(kind), dA, zero(dB).to(kind), zero(dC).to(kind), dD, dz.to(kind),
            ddt.sum((0, 1), dtype=torch.float64).float()]
    if s["case"]["state"]:
        out.append(back[:, 0].clone())
    return tuple(out)


_PLAIN = {"norm": _norm, "conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _exact_norm(t, case):
    x, w = t["x"], t["weight"]
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    hat = (x - mean) / (var + 1e-5).sqrt()
    y = hat * w + t["bias"]
    if not case["grad"]:
        return (y,)
    g, n = t["dy"] * w, x.shape[1]
    # dx = J^T g with J = (I - 1/n - hat hat^T / n) / sqrt(var + eps)
    dx = (g - g.sum(1, keepdim=True) / n - hat * ((g * hat).sum(1, keepdim=True) / n)) / (var + 1e-5).sqrt()
    return y, dx, (t["dy"] * hat).sum(0), t["dy"].sum(0)


def _exact_conv(t, case):
    """Position by position: an input's share in each output that its window reaches."""
    x, w = t["x"], t["weight"]
    b, length, e = x.shape
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    head = t.get("state", torch.zeros(b, _K - 1, e, dtype=x.dtype, device=x.device))
    dhead, dw, db = torch.zeros_like(head), torch.zeros_like(w), torch.zeros_like(t["bias"])
    ends = t["lens"].tolist() if "lens" in t else [length] * b
    final = torch.empty_like(head)
    for i in range(b):
        n = ends[i]
        row = torch.cat([head[i], x[i, :n]])
        p = t["bias"].expand(n, e).clone()
        for k in range(_K):
            p += w[:, k] * row[k:k + n]
        y[i, :n] = p * torch.sigmoid(p)
        final[i] = row[n:]
        if case["grad"]:
            sig = torch.sigmoid(p)
            dp = t["dy"][i, :n] * (sig + p * sig * (1 - sig))
            drow = torch.zeros_like(row)
            if case["state"]:
                drow[n:] = t["dstate"][i]
            for k in range(_K):
                drow[k:k + n] += w[:, k] * dp
                dw[:, k] += (dp * row[k:k + n]).sum(0)
            db += dp.sum(0)
            dx[i, :n], dhead[i] = drow[_K - 1:], drow[:_K - 1]
    out = [y] + ([final] if case["state"] else [])
    if case["grad"]:
        out += [dx, dw, db] + ([dhead] if case["state"] else [])
    return tuple(out)


def _exact_conv_step(t, case):
    row = torch.cat([t["state"], t["x"][:, None]], 1)
    p = t["bias"] + sum(row[:, k] * t["weight"][:, k] for k in range(_K))
    return p * torch.sigmoid(p), row[:, 1:]


def _exact_scan(t, case):
    """Token by token, forwards and then backwards."""
    x, A, D = t["x"], t["A"], t["D"]
    b, length, e = x.shape
    dt = t["dt"] + t["dt_bias"]
    d = torch.logaddexp(dt, torch.zeros_like(dt))
    live = torch.ones(b, length, dtype=torch.bool, device=x.device)
    if "lens" in t:
        live = torch.arange(length, device=x.device)[None] < t["lens"][:, None]
    d = d * live[..., None]
    h = t["state"].clone() if "state" in t else torch.zeros(b, e, _N, dtype=x.dtype, device=x.device)
    first = h
    kept = []
    v = torch.zeros_like(x)
    for i in range(length):
        h = h * torch.exp(d[:, i, :, None] * A) + (d[:, i] * x[:, i])[..., None] * t["B"][:, i, None]
        v[:, i] = (h * t["C"][:, i, None]).sum(-1)
        if case["grad"]:
            kept.append(h)
    v = v + D * x
    sig = torch.sigmoid(t["z"])
    y = v * t["z"] * sig * live[..., None]
    out = [y] + ([h] if case["state"] else [])
    if not case["grad"]:
        return tuple(out)
    dy = t["dy"] * live[..., None]
    g = dy * t["z"] * sig
    dz = dy * v * (sig + t["z"] * sig * (1 - sig))
    dx, ddt, dB, dC = D * g, torch.zeros_like(x), torch.zeros_like(t["B"]), torch.zeros_like(t["C"])
    dA = torch.zeros_like(A)
    dh = t["dstate"].clone() if case["state"] else torch.zeros_like(h)
    for i in reversed(range(length)):
        a = torch.exp(d[:, i, :, None] * A)
        h, prev = kept[i], kept[i - 1] if i else first
        dC[:, i] = (g[:, i, :, None] * h).sum(1)
        dh = dh + g[:, i, :, None] * t["C"][:, i, None]
        dB[:, i] = ((d[:, i] * x[:, i])[..., None] * dh).sum(1)
        into = (dh * t["B"][:, i, None]).sum(-1)
        dx[:, i] += into * d[:, i]
        dh = dh * a
        grow = dh * prev
        ddt[:, i] = into * x[:, i] + (grow * A).sum(-1)
        dA += (grow * d[:, i, :, None]).sum(0)
    ddt = ddt * torch.sigmoid(dt) * live[..., None]
    dB, dC = dB * live[..., None], dC * live[..., None]
    out += [dx * live[..., None], ddt, dA, dB, dC, (g * x).sum((0, 1)), dz, ddt.sum((0, 1))]
    return tuple(out + ([dh] if case["state"] else []))


def _exact_scan_step(t, case):
    dt = t["dt"] + t["dt_bias"]
    d = torch.logaddexp(dt, torch.zeros_like(dt))
    h = t["state"] * torch.exp(d[:, :, None] * t["A"]) + (d * t["x"])[:, :, None] * t["B"][:, None, :]
    v = torch.einsum("ben,bn->be", h, t["C"]) + t["D"] * t["x"]
    return v * t["z"] * torch.sigmoid(t["z"]), h


_EXACT = {"norm": _exact_norm, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
          "scan_step": _exact_scan_step}


def exact(case, seed):
    s = prepare(case, seed)
    t = {k: v.detach().double() if v.is_floating_point() else v for k, v in s.items() if isinstance(v, torch.Tensor)}
    with torch.no_grad():
        return _EXACT[case["op"]](t, case)
