"""Refusals of pointers that a kernel could not load from, without a GPU: they
end in an error code before anything is launched."""
import ctypes

from boa_b200 import _native as _n


def test_layer_norm_statistics_alignment():
    """mean and 1/sigma of a row move as one 8-byte access."""
    lib = _n.load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 4)
    rc = lib.boa_layer_norm(4, 8, 0, p, 8, p, p, 1e-5, p, odd, 0, None)
    assert rc == _n.BOA_ERR_ARG and "8-byte aligned" in lib.boa_last_error().decode()
    rc = lib.boa_layer_norm_backward(4, 8, 0, p, 8, p, 8, p, odd, p, p, p, p, 1 << 20, 0, None)
    assert rc == _n.BOA_ERR_ARG and "8-byte aligned" in lib.boa_last_error().decode()
