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
