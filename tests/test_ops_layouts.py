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
