"""boa_b200.ops without a GPU: refusals of the Python and C entry points, the
argument structs' layout, and the references' gradients."""
import ctypes
import os
import subprocess

import pytest
import torch

import ops_reference as ref
from boa_b200 import _native as _n
from boa_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _scan_inputs(b=2, length=5, e=8, kind=torch.float32):
    z = lambda *s: torch.zeros(*s, dtype=kind)  # noqa: E731
    return [z(b, length, e), z(b, length, e), torch.zeros(e, 16), z(b, length, 16), z(b, length, 16), torch.zeros(e),
            z(b, length, e), torch.zeros(e)]


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layer_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.causal_conv_step(x[:, 0], torch.zeros(2, 3, 8), torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.ssm_scan(*_scan_inputs())
    a = _scan_inputs()
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.ssm_step(a[0][:, 0], a[1][:, 0], torch.zeros(2, 8, 16), a[2], a[3][:, 0], a[4][:, 0])


def test_layer_norm_refusals():
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        ops.layer_norm(torch.zeros(2, 8, dtype=torch.float64), torch.ones(8))
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(torch.zeros(2, 8), torch.ones(7))
    with pytest.raises(ValueError, match="bias"):
        ops.layer_norm(torch.zeros(2, 8), torch.ones(8), torch.ones(2, 8))
    with pytest.raises(ValueError, match="at least one"):
        ops.layer_norm(torch.zeros(2, 0), torch.ones(0))
    with pytest.raises(ValueError, match="at least one"):
        ops.layer_norm(torch.tensor(1.0), torch.ones(1))


def test_causal_conv_refusals():
    x = torch.zeros(2, 5, 8)
    for w in (torch.zeros(8, 1), torch.zeros(8, 5), torch.zeros(7, 4), torch.zeros(8, 2, 4)):
        with pytest.raises(ValueError, match="weight"):
            ops.causal_conv(x, w)
    w = torch.zeros(8, 4)
    with pytest.raises(ValueError, match=r"\[batch, length, channels\]"):
        ops.causal_conv(x[0], w)
    with pytest.raises(ValueError, match="bias"):
        ops.causal_conv(x, w, torch.zeros(4))
    with pytest.raises(ValueError, match="state"):
        ops.causal_conv(x, w, state=torch.zeros(2, 4, 8))
    with pytest.raises(ValueError, match="type of x"):
        ops.causal_conv(x, w, state=torch.zeros(2, 3, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="lens"):
        ops.causal_conv(x, w, lens=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="lens"):
        ops.causal_conv(x, w, lens=torch.zeros(2))
    with pytest.raises(ValueError, match="contiguous"):
        ops.causal_conv_step(x[:, 0], torch.zeros(2, 8, 3).transpose(1, 2), w)
    with pytest.raises(ValueError, match=r"\[batch, channels\]"):
        ops.causal_conv_step(x, torch.zeros(2, 3, 8), w)


@pytest.mark.parametrize("i,name,bad", [
    (0, "x", torch.zeros(5, 8)), (0, "x", torch.zeros(2, 5, 8, dtype=torch.int32)), (1, "dt", torch.zeros(2, 4, 8)),
    (2, "A", torch.zeros(8, 8)), (2, "A", torch.zeros(16)), (3, "B", torch.zeros(2, 5, 8)),
    (4, "C", torch.zeros(2, 5, 1, 16)), (5, "D", torch.zeros(9)), (6, "z", torch.zeros(2, 5, 7)),
    (7, "dt_bias", torch.zeros(1)), (1, "dt", torch.zeros(2, 5, 8, dtype=torch.float16)),
    (6, "z", torch.zeros(2, 5, 8, dtype=torch.bfloat16))])
def test_ssm_scan_refusals(i, name, bad):
    a = _scan_inputs()
    a[i] = bad
    with pytest.raises(ValueError, match=name):
        ops.ssm_scan(*a)


def test_ssm_state_refusals():
    a = _scan_inputs()
    with pytest.raises(ValueError, match="state"):
        ops.ssm_scan(*a, state=torch.zeros(2, 16, 8))
    with pytest.raises(ValueError, match="float32"):
        ops.ssm_scan(*a, state=torch.zeros(2, 8, 16, dtype=torch.bfloat16))
    s = [a[0][:, 0], a[1][:, 0], None, a[2], a[3][:, 0], a[4][:, 0]]
    for bad in (torch.zeros(2, 16, 8).transpose(1, 2), torch.zeros(2 * 8 * 16 + 1)[1:].view(2, 8, 16),
                torch.zeros(1, 8, 16).expand(2, 8, 16)):
        s[2] = bad
        with pytest.raises(ValueError, match="contiguous"):
            ops.ssm_step(*s)


def test_sizes_beyond_32_bits_are_refused():
    wide = torch.zeros(1, 1, 1).expand(2 ** 31, 1, 1)
    with pytest.raises(ValueError, match="below 2"):
        ops.causal_conv(wide, torch.zeros(1, 4))
    with pytest.raises(ValueError, match="below 2"):
        ops.layer_norm(wide[:, 0, 0], torch.zeros(1))
    with pytest.raises(ValueError, match="below 2"):
        ops.ssm_scan(wide, wide, torch.zeros(1, 16), wide.expand(-1, -1, 16), wide.expand(-1, -1, 16))


def test_not_a_tensor():
    with pytest.raises(TypeError, match="weight must be a tensor"):
        ops.layer_norm(torch.zeros(2, 8), None)
    with pytest.raises(TypeError, match="x must be a tensor"):
        ops.causal_conv([1.0], torch.zeros(8, 4))


def test_struct_layout_matches_header(tmp_path):
    """Field offsets and sizes of the ctypes structs are the C compiler's."""
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "boa_b200.h"', "int main(void) {"]
    want = []
    for cname, cls in (("boa_conv_args", _n.ConvArgs), ("boa_ssm_args", _n.SsmArgs)):
        src.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            src.append(f'  printf("%zu\\n", offsetof({cname}, {f}));')
            want.append(getattr(cls, f).offset)
    src.append("  return 0;\n}")
    (tmp_path / "t.c").write_text("\n".join(src))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "t")]).split()]
    assert got == want


def _refused(rc, code, text):
    assert rc == code
    assert text in _n.load().boa_last_error().decode()


def test_c_entry_points_refuse():
    """Bad arguments end in an error code before anything is launched."""
    lib = _n.load()
    assert lib.boa_layer_norm(0, 8, 0, None, 8, None, None, 1e-5, None, None, 0, None) == _n.BOA_OK
    _refused(lib.boa_layer_norm(4, 8, 0, None, 8, None, None, 1e-5, None, None, 0, None), _n.BOA_ERR_ARG, "null")
    _refused(lib.boa_layer_norm(4, 0, 0, None, 8, None, None, 1e-5, None, None, 0, None), _n.BOA_ERR_ARG, "width")
    _refused(lib.boa_layer_norm(4, 8193, 0, None, 8, None, None, 1e-5, None, None, 0, None), _n.BOA_ERR_UNSUPPORTED,
             "8192")
    _refused(lib.boa_layer_norm(4, 8, 3, None, 8, None, None, 1e-5, None, None, 0, None), _n.BOA_ERR_ARG, "dtype")
    assert lib.boa_layer_norm_workspace_bytes(4, 8193, 0) == 0
    p = ctypes.c_void_p(64)
    _refused(lib.boa_layer_norm_backward(4, 8, 0, p, 8, p, 8, p, p, p, p, p, None, 0, 0, None), _n.BOA_ERR_ARG,
             "workspace")
    _refused(lib.boa_causal_conv(None, None), _n.BOA_ERR_ARG, "null")
    a = _n.ConvArgs(batch=1, length=4, channels=8, width=5)
    _refused(lib.boa_causal_conv(ctypes.byref(a), None), _n.BOA_ERR_UNSUPPORTED, "width")
    a.width = 4
    _refused(lib.boa_causal_conv(ctypes.byref(a), None), _n.BOA_ERR_ARG, "null")
    _refused(lib.boa_causal_conv_step(ctypes.byref(a), None), _n.BOA_ERR_ARG, "null")
    a.x = a.dy = a.dx = a.weight = a.dweight = 64
    _refused(lib.boa_causal_conv_backward(ctypes.byref(a), None), _n.BOA_ERR_ARG, "workspace")
    a.batch = -1
    _refused(lib.boa_causal_conv(ctypes.byref(a), None), _n.BOA_ERR_ARG, "batch")
    s = _n.SsmArgs(batch=1, length=100, channels=8, states=8)
    _refused(lib.boa_ssm_scan(ctypes.byref(s), None), _n.BOA_ERR_UNSUPPORTED, "states")
    s.states = 16
    _refused(lib.boa_ssm_scan(ctypes.byref(s), None), _n.BOA_ERR_ARG, "null")
    _refused(lib.boa_ssm_step(ctypes.byref(s), None), _n.BOA_ERR_ARG, "null")
    s.A = s.x = s.dt = s.B = s.C = s.y = s.dy = s.dx = s.ddt = s.dB = s.dC = s.dA = s.checkpoints = 64
    _refused(lib.boa_ssm_scan(ctypes.byref(s), None), _n.BOA_ERR_ARG, "workspace")
    _refused(lib.boa_ssm_scan_backward(ctypes.byref(s), None), _n.BOA_ERR_ARG, "workspace")
    s.state_out = 68
    _refused(lib.boa_ssm_step(ctypes.byref(s), None), _n.BOA_ERR_ARG, "aligned")
    s.dtype = 7
    _refused(lib.boa_ssm_scan(ctypes.byref(s), None), _n.BOA_ERR_ARG, "dtype")


# The references' hand-written gradients against autograd in 64 bits.
def test_reference_gradients():
    g = torch.Generator()
    g.manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dy = r(6, 10), r(10), r(10), r(6, 10)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (10,), leaves[1], leaves[2])
    vals, _ = ref.norm(x, w, b, dy)
    for a, v in zip((y,) + torch.autograd.grad(y, leaves, dy), vals):
        assert torch.allclose(a, v, rtol=1e-10, atol=1e-10)

    lens = torch.tensor([7, 0, 4])
    x, w, b, s, dy, ds = r(3, 7, 5), r(5, 4), r(5), r(3, 3, 5), r(3, 7, 5), r(3, 3, 5)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, s)]
    live = (torch.arange(7)[None] < lens[:, None])[..., None]
    full = torch.cat([leaves[3], leaves[0]], 1)
    p = leaves[2] + sum(leaves[1][:, k] * full[:, k:k + 7] for k in range(4))
    y = torch.nn.functional.silu(p) * live
    out = torch.stack([full[i, n:n + 3] for i, n in enumerate(lens.tolist())])
    got = ref.conv(x, w, b, True, s, lens, dy, ds)
    for name, a in zip(("y", "state", "dx", "dw", "db", "dstate"),
                       (y, out) + torch.autograd.grad((y, out), leaves, (dy, ds))):
        assert torch.allclose(a, got[name][0], rtol=1e-10, atol=1e-10), name

    x, dt, B, C, z, dy = r(3, 7, 5), r(3, 7, 5), r(3, 7, 16), r(3, 7, 16), r(3, 7, 5), r(3, 7, 5)
    A, D, bias, s, ds = -torch.exp(r(5, 16)), r(5), r(5), r(3, 5, 16), r(3, 5, 16)
    leaves = [t.clone().requires_grad_() for t in (x, dt, A, B, C, D, z, bias, s)]
    lx, ldt, lA, lB, lC, lD, lz, lb, h = leaves
    d, ys = torch.nn.functional.softplus(ldt + lb) * live, []
    for t in range(7):
        h = torch.exp(d[:, t, :, None] * lA) * h + (d[:, t] * lx[:, t])[..., None] * lB[:, t, None]
        ys.append((h * lC[:, t, None]).sum(-1) + lD * lx[:, t])
    y = torch.stack(ys, 1) * torch.nn.functional.silu(lz) * live
    got = ref.scan(x, dt, A, B, C, D, z, bias, True, s, lens, dy, ds)
    for name, a in zip(("y", "state", "dx", "ddt", "dA", "dB", "dC", "dD", "dz", "dbias", "dstate"),
                       (y, h) + torch.autograd.grad((y, h), leaves, (dy, ds))):
        assert torch.allclose(a, got[name][0], rtol=1e-10, atol=1e-10), name
