"""Calls of the C entry points from two host threads at once, each on its own
stream with its own memory: kernels of one template that want different
amounts of shared memory."""
import ctypes
import threading

import pytest
import torch

from boa_b200 import _native as _n

pytestmark = pytest.mark.gpu
TIMES = 400


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _at_once(calls):
    """Every call TIMES times in a thread of its own; the errors."""
    errors, start = [], threading.Barrier(len(calls))

    def work(call, stream):
        start.wait()
        for _ in range(TIMES):
            rc = call(ctypes.c_void_p(stream.cuda_stream))
            if rc != _n.BOA_OK:
                errors.append((rc, _n.load().boa_last_error().decode()))
                return

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(c, torch.cuda.Stream())) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


def _scan_backward(E, keep):
    """A backward call of [1, 8, E] and its dA, behind one forward call."""
    lib = _n.load()
    g = torch.Generator(device="cuda").manual_seed(E)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = {k: r(1, 8, E) for k in ("x", "dt", "dy")}
    t.update({k: torch.empty(1, 8, E, device="cuda") for k in ("y", "dx", "ddt")})
    t.update({k: r(1, 8, 16) for k in ("B", "C", "dB", "dC")})
    t.update(A=-torch.rand(E, 16, generator=g, device="cuda"), dA=torch.empty(E, 16, device="cuda"))
    a = _n.SsmArgs(batch=1, length=8, channels=E, states=16, softplus=1, device=0, x_bs=8 * E, x_ts=E, dt_bs=8 * E,
                   dt_ts=E, B_bs=128, B_ts=16, C_bs=128, C_ts=16, dy_bs=8 * E, dy_ts=E)
    sizes = {"checkpoints": lib.boa_ssm_checkpoint_bytes(ctypes.byref(a)),
             "workspace": max(lib.boa_ssm_workspace_bytes(ctypes.byref(a), b) for b in (0, 1))}
    t.update({k: torch.empty(n, dtype=torch.uint8, device="cuda") for k, n in sizes.items()})
    for k, v in t.items():
        setattr(a, k, v.data_ptr())
    a.workspace_bytes = sizes["workspace"]
    assert lib.boa_ssm_scan(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == _n.BOA_OK
    keep.append((t, a))
    return (lambda s: lib.boa_ssm_scan_backward(ctypes.byref(a), s)), t["dA"]


def test_scan_backward_of_different_widths():
    keep = []
    made = [_scan_backward(E, keep) for E in (512, 64, 512, 192)]
    want = []
    for call, dA in made:
        assert call(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == _n.BOA_OK
        torch.cuda.synchronize()
        want.append(dA.clone())
        dA.zero_()
    assert _at_once([c for c, _ in made]) == []
    assert all(torch.equal(dA, w) for (_, dA), w in zip(made, want))


def test_layer_norm_backward_of_different_widths():
    lib = _n.load()
    keep = []

    def make(width):
        x, dy, dx = (torch.randn(4, width, device="cuda") for _ in range(3))
        w, dw, db = (torch.ones(width, device="cuda") for _ in range(3))
        stats = torch.ones(4, 2, device="cuda")
        ws = torch.empty(lib.boa_layer_norm_workspace_bytes(4, width, 0), dtype=torch.uint8, device="cuda")
        keep.append((x, dy, dx, w, dw, db, stats, ws))
        return lambda s: lib.boa_layer_norm_backward(4, width, 0, _p(x), width, _p(dy), width, _p(w), _p(stats), _p(dx),
                                                     _p(dw), _p(db), _p(ws), ws.numel(), 0, s)

    assert _at_once([make(w) for w in (8192, 6400, 8000, 6208)]) == []
