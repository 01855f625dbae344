"""boa_b200.ops under torch's other ways to run a function: each either gives
the right result or is refused, without a GPU as far as the refusals go."""
import pytest
import torch
from torch.autograd import forward_ad

from boa_b200 import ops

B, L, E = 2, 5, 8


def _inputs():
    """{call: (function, its floating inputs)} on the CPU, where nothing can be launched."""
    r = lambda *s: torch.randn(*s)  # noqa: E731
    scan = [r(B, L, E), r(B, L, E), -torch.rand(E, 16), r(B, L, 16), r(B, L, 16), r(E), r(B, L, E), r(E)]
    step = [t[:, 0] if t.dim() == 3 else t for t in scan]
    return {
        "layer_norm": (lambda x, w, b: ops.layer_norm(x, w, b), [r(B, E), r(E), r(E)]),
        "causal_conv": (lambda x, w, b, s: ops.causal_conv(x, w, b, state=s), [r(B, L, E), r(E, 4), r(E), r(B, 3, E)]),
        "causal_conv_step": (lambda x, s, w, b: ops.causal_conv_step(x, s, w, b),
                             [r(B, E), r(B, 3, E), r(E, 4), r(E)]),
        "ssm_scan": (lambda *a: ops.ssm_scan(*a[:8], state=a[8]), scan + [r(B, E, 16)]),
        "ssm_step": (lambda *a: ops.ssm_step(a[0], a[1], a[8], *a[2:8]), step + [r(B, E, 16)]),
    }


@pytest.mark.parametrize("name", ["layer_norm", "causal_conv", "causal_conv_step", "ssm_scan", "ssm_step"])
def test_forward_mode_tangents_are_refused(name):
    """A tangent on any floating input: the result would come back without one, which reads as a zero derivative."""
    f, inputs = _inputs()[name]
    for i in range(len(inputs)):
        with forward_ad.dual_level():
            a = list(inputs)
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*a)
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                f(*a)
            # a mode without tangents takes the tensor for what it is (and then finds it on the CPU)
            with pytest.raises(RuntimeError, match="no CPU path"), torch.inference_mode():
                f(*a)


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_in_backward():
    """Forward over reverse: a tangent on the incoming gradient or on a saved input."""
    for name in ("layer_norm", "causal_conv", "ssm_scan"):
        f, inputs = _inputs()[name]
        a = [t.cuda() for t in inputs]
        a[0].requires_grad_()
        y = f(*a)
        with forward_ad.dual_level():
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, a[0], dy, retain_graph=True)
        assert torch.isfinite(torch.autograd.grad(y, a[0], torch.ones_like(y))[0]).all()


@pytest.mark.parametrize("name", ["layer_norm", "causal_conv", "causal_conv_step", "ssm_scan", "ssm_step"])
@pytest.mark.parametrize("grad", [False, True])
def test_tracing_is_refused(name, grad):
    """torch.jit.trace would record the result as a constant and the traced function would ignore its input."""
    f, inputs = _inputs()[name]
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, tuple(inputs))


# ------------------------------------------------------------------- values that are not finite, behind a row's end
@pytest.mark.gpu
@pytest.mark.parametrize("E", [24, 33])
def test_scan_gradients_behind_a_row_are_zero_whatever_the_rest_holds(E):
    """D, the gradient of the final state or A of inf or NaN reach the tokens of a row, not those behind its end."""
    g = torch.Generator().manual_seed(E)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    lens = torch.tensor([0, 3, 11, 16, 17], device="cuda")
    leaves = [r(5, 18, E), r(5, 18, E), r(5, 18, 16), r(5, 18, 16), r(5, 18, E)]
    A, D, dout = -torch.rand(E, 16, generator=g).cuda(), r(E), r(5, E, 16)
    A[3], D[::2], dout[:, 5] = float("nan"), float("inf"), float("inf")
    x, dt, B, C, z = (t.requires_grad_() for t in leaves)
    y, out = ops.ssm_scan(x, dt, A, B, C, D, z, lens=lens, return_state=True)
    grads = torch.autograd.grad((y, out), (x, dt, B, C, z), (r(5, 18, E), dout))
    behind = torch.arange(18, device="cuda") >= lens[:, None]
    for name, t in zip(("y", "dx", "ddt", "dB", "dC", "dz"), (y,) + grads):
        assert (t[behind] == 0).all(), name


@pytest.mark.gpu
def test_scan_channels_that_forget_at_once():
    """A of -inf: the decay is 0 at every token and 1 behind a row's end, forward, backward and for single tokens."""
    import ops_reference as ref
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    nb, length, e = 3, 21, 24
    x, dt, z, dy = (r(nb, length, e) for _ in range(4))
    B, C = r(nb, length, 16), r(nb, length, 16)
    A, D, bias, state, dout = -torch.rand(e, 16, generator=g), r(e), r(e), r(nb, e, 16), r(nb, e, 16)
    A[::3], A[1, 4] = float("-inf"), float("-inf")
    lens = torch.tensor([21, 1, 13], dtype=torch.int32)
    # in the reference a decay that is 0 from the smallest d on, but with a product of 0 behind the row
    far = torch.where(A == float("-inf"), torch.tensor(-1e30), A)
    want = ref.scan(*[t.double() for t in (x, dt, far, B, C, D, z, bias)], True, state.double(), lens, dy.double(),
                    dout.double())
    names = ("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "dbias", "dstate")
    leaves = [t.cuda().requires_grad_() for t in (x, dt, A, B, C, D, z, bias, state)]
    y, out = ops.ssm_scan(*leaves[:8], state=leaves[8], lens=lens.cuda(), return_state=True)
    grads = torch.autograd.grad((y, out), leaves, (dy.cuda(), dout.cuda()))
    # counts of the scan's own tests: 8 a token and 64, twice and more where two such results meet or rows are summed
    for name, t in zip(("y", "state") + names, (y, out) + grads):
        ref.close(name, t, *want[name], 16 * length + 128 + nb * length / 8)
    st = state.cuda()
    with torch.no_grad():
        one = ops.ssm_step(x[:, 0].cuda(), torch.full((nb, e), -200.0).cuda(), st, A.cuda(), B[:, 0].cuda(), C[:, 0].cuda())
    assert torch.equal(st, state.cuda()) and torch.isfinite(one).all()      # d underflows to 0: nothing moves


@pytest.mark.gpu
def test_scan_split_over_states_that_grow():
    """A above 0: a part's decay overflows fp32 (e^3 a token) while the state that enters it is still 0, which is then
    0 behind it too.  Only the last 16 tokens of a row have an input, so no value of the definition leaves fp32."""
    import ops_reference as ref
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    length, e = 1200, 8
    x, dt = r(2, length, e), 3.0 + 0.1 * r(2, length, e)
    lens = torch.tensor([length, 700], dtype=torch.int32)
    for i, n in enumerate(lens.tolist()):
        x[i, :n - 16] = 0.0
    B, C, A = r(2, length, 16), r(2, length, 16), torch.ones(e, 16)
    want = ref.scan(*[t.double() for t in (x, dt, A, B, C)], None, None, None, True, None, lens, torch.zeros_like(x).double(),
                    None)
    with torch.no_grad():
        y, h = ops.ssm_scan(*[t.cuda() for t in (x, dt, A, B, C)], lens=lens.cuda(), return_state=True)
    # 16 tokens, each with an exponent of up to 4.7 whose 3 roundings the decay scales by 3.3, and 5 more; and 96 at the end
    ref.close("y", y, *want["y"], 16 * 15 + 96)
    ref.close("state", h, *want["state"], 16 * 15 + 64)
