"""The block operators at the ends of their 32-bit sizes."""
import ctypes

import pytest
import torch

from boa_b200 import _native as _n

F32, BF16 = torch.float32, torch.bfloat16
MOST = 2 ** 31 - 1 - 2 ** 16


def _ops():
    from boa_b200 import ops
    return ops


def test_sizes_that_would_overflow_are_refused():
    """Refused by the library before anything is launched; the largest sizes pass this check (and end at the next)."""
    lib = _n.load()

    def end(call, args):
        rc = getattr(lib, call)(ctypes.byref(args), None)
        return rc, lib.boa_last_error().decode()

    for call in ("boa_causal_conv", "boa_causal_conv_backward", "boa_causal_conv_step"):
        for length, channels in ((MOST + 1, 1), (2 ** 31 - 1, 1), (1, MOST + 1), (1, 2 ** 31 - 1)):
            rc, why = end(call, _n.ConvArgs(batch=1, length=length, channels=channels, width=4))
            assert rc == _n.BOA_ERR_UNSUPPORTED and "2^31 - 2^16" in why
        rc, why = end(call, _n.ConvArgs(batch=1, length=MOST, channels=MOST, width=4))
        assert rc == _n.BOA_ERR_ARG and "null" in why
    for call in ("boa_ssm_scan", "boa_ssm_scan_backward", "boa_ssm_step"):
        for length, channels in ((MOST + 1, 1), (2 ** 31 - 1, 1), (1, MOST + 1), (1, 2 ** 31 - 1)):
            rc, why = end(call, _n.SsmArgs(batch=1, length=length, channels=channels, states=16))
            assert rc == _n.BOA_ERR_UNSUPPORTED and "2^31 - 2^16" in why
        rc, why = end(call, _n.SsmArgs(batch=1, length=MOST, channels=MOST, states=16))
        assert rc == _n.BOA_ERR_ARG and "null" in why


@pytest.mark.parametrize("length,channels", [(MOST, 1), (MOST, 33), (1, MOST), (2 ** 28, 7)])
def test_workspace_sizes_do_not_wrap(length, channels):
    """A row of partial sums for every block: never less than one row of (width + 1) or 18 floats a channel, and never
    more than the blocks of eight rounds need."""
    lib = _n.load()
    got = lib.boa_causal_conv_workspace_bytes(ctypes.byref(
        _n.ConvArgs(batch=1, length=length, channels=channels, width=4)))
    assert 5 * channels * 4 <= got <= 296 * 5 * channels * 4
    a = _n.SsmArgs(batch=1, length=length, channels=channels, states=16)
    assert lib.boa_ssm_checkpoint_bytes(ctypes.byref(a)) == (length + 7) // 8 * channels * 64
    groups = -(-channels // 512)
    sums = 128 * groups * length if groups > 1 else 0
    got = lib.boa_ssm_workspace_bytes(ctypes.byref(a), 1)
    assert 72 * channels <= got - sums <= (72 + 68) * channels * 148 * 8 + 16
    forward = lib.boa_ssm_workspace_bytes(ctypes.byref(a), 0)
    assert forward <= 68 * channels * (1776 + 1)
    if channels <= 33:                       # a long row of few channels is split over its length, both ways
        assert forward >= 68 * channels * 880 and got - sums >= 140 * channels * 70


# Channels repeat a short pattern, so that every repeat has to give the bits of a call on the pattern alone.
PATTERN = 4096


def _repeated(small, n):
    """small [.., PATTERN, ..] on the first axis, n times."""
    out = torch.empty((n,) + tuple(small.shape), dtype=small.dtype, device="cuda")
    out.copy_(small)
    return out.flatten(0, 1)


def _repeats(big, small):
    return bool((big.view((-1,) + tuple(small.shape)) == small).all())


@pytest.mark.gpu
def test_scan_with_more_channel_sums_than_32_bits():
    """18 sums a channel: 2^28 channels have more than 2^32 of them."""
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    n = 2 ** 28 // PATTERN
    small = {"x": r(PATTERN).to(BF16), "dt": r(PATTERN).to(BF16), "A": -torch.rand(PATTERN, 16, device="cuda"),
             "D": r(PATTERN), "bias": r(PATTERN), "dy": r(PATTERN).to(BF16)}
    B, C = r(1, 1, 16).to(BF16), r(1, 1, 16).to(BF16)

    def run(t):
        leaves = [t[k].requires_grad_() for k in ("A", "D", "bias")]
        y = _ops().ssm_scan(t["x"][None, None], t["dt"][None, None], t["A"], B, C, t["D"], None, t["bias"])
        return (y.detach()[0, 0],) + torch.autograd.grad(y, leaves, t["dy"][None, None])

    want = run({k: v.clone() for k, v in small.items()})
    got = run({k: _repeated(v, n) for k, v in small.items()})
    for name, a, b in zip(("y", "dA", "dD", "dbias"), got, want):
        assert _repeats(a, b), name
    del got
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_convolution_with_more_channel_sums_than_32_bits():
    """5 sums a channel: 2^29 channels have more than 2^31 of them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    small = {"x": r(PATTERN).to(BF16), "w": r(PATTERN, 4), "b": r(PATTERN), "dy": r(PATTERN).to(BF16)}

    def run(t):
        leaves = [t[k].requires_grad_() for k in ("x", "w", "b")]
        y = _ops().causal_conv(t["x"][None, None], t["w"], t["b"])
        return (y.detach()[0, 0],) + torch.autograd.grad(y, leaves, t["dy"][None, None])

    want = run({k: v.clone() for k, v in small.items()})
    got = run({k: _repeated(v, 2 ** 29 // PATTERN) for k, v in small.items()})
    for name, a, b in zip(("y", "dx", "dw", "db"), got, want):
        assert _repeats(a, b), name
    del got
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_scan_step_with_more_threads_a_row_than_32_bits():
    """4 threads a channel: 2^29 channels."""
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    small = {"x": r(PATTERN).to(BF16), "dt": r(PATTERN).to(BF16), "A": -torch.rand(PATTERN, 16, device="cuda"),
             "state": r(PATTERN, 16)}
    B, C = r(1, 16).to(BF16), r(1, 16).to(BF16)

    def run(t):
        with torch.no_grad():
            return _ops().ssm_step(t["x"][None], t["dt"][None], t["state"][None], t["A"], B, C)[0], t["state"]

    want = run({k: v.clone() for k, v in small.items()})
    got = run({k: _repeated(v, 2 ** 29 // PATTERN) for k, v in small.items()})
    assert _repeats(got[0], want[0]) and _repeats(got[1], want[1])
    del got
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_longest_convolution():
    """One channel of MOST tokens; its end against a call on the last tokens alone, outputs and gradients."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1, MOST, 1, generator=g, device="cuda", dtype=BF16).requires_grad_()
    w = torch.randn(1, 4, generator=g, device="cuda").requires_grad_()
    dy = torch.zeros(1, 1, 1, device="cuda", dtype=BF16).expand(1, MOST, 1).contiguous()
    dy[:, -300:] = torch.randn(1, 300, 1, generator=g, device="cuda", dtype=BF16)
    y = _ops().causal_conv(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    last = x[:, -303:].detach().clone().requires_grad_()
    yl = _ops().causal_conv(last, w)
    dxl, dwl = torch.autograd.grad(yl, (last, w), dy[:, -303:].contiguous())
    assert torch.equal(y[:, -300:], yl[:, 3:]) and torch.equal(dx[:, -303:], dxl)
    # the same 300 products (each off by at most 64 roundings and none apart) summed in two orders: 300 roundings each
    # of the sum of |dp x| <= |dy| (1.1 + |p| / 2) |x|
    size = (dy[:, -300:].float().abs() * (1.1 + 2 * w.abs().sum())).sum() * last.abs().max()
    assert ((dw - dwl).abs() <= 2 * 364 * 2.0 ** -24 * size).all() and (dw != 0).any()
    assert not dx[:, :MOST - 303].any()
    del y, dx, dy, x
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_longest_scan():
    """One channel of MOST tokens whose decays forget within a hundred of them; its end against a call on the last
    4096 alone.  The two split the length differently.  A token passes 8 roundings and is then halved at least, so a
    state is off by 16 of them, and 64 + 32 more for softplus and the sum over states: 112 on each side, of the same
    sums of absolute values; the bf16 results may then be rounded to neighbours."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(1, MOST, 1, generator=g, device="cuda", dtype=BF16)
    dt = torch.rand(1, MOST, 1, generator=g, device="cuda", dtype=BF16)
    A = -1.0 - torch.rand(1, 16, generator=g, device="cuda")
    B, C = (torch.randn(1, 1, 16, generator=g, device="cuda").to(BF16) for _ in range(2))
    n = 4096
    with torch.no_grad():
        y, h = _ops().ssm_scan(x, dt, A, B.expand(1, MOST, 16), C.expand(1, MOST, 16), return_state=True)
        yl, hl = _ops().ssm_scan(x[:, -n:], dt[:, -n:], A, B.expand(1, n, 16), C.expand(1, n, 16), return_state=True)
        s, hs = _ops().ssm_scan(x[:, -n:].float().abs(), dt[:, -n:].float(), A, B.expand(1, n, 16).float().abs(),
                                C.expand(1, n, 16).float().abs(), return_state=True)
    # d >= softplus(0) = 0.69 and A <= -1: what is 200 tokens old has decayed by 2^-200
    a, b, fp32 = y[0, 200 - n:, 0].double(), yl[0, 200:, 0].double(), 224 * 2.0 ** -24 * s[0, 200:, 0].double()
    assert ((a - b).abs() <= fp32 + torch.finfo(BF16).eps * (b.abs() + fp32)).all()
    assert ((h - hl).abs() <= 224 * 2.0 ** -24 * hs).all()
    assert a.any()
    del y, x, dt
    torch.cuda.empty_cache()
