"""Operators of a Mamba block outside its matrix products, on the sm_100a
kernels of libboa_b200.so (``boa_layer_norm``, ``boa_causal_conv``,
``boa_ssm_scan`` and their backward and one-token forms):

* ``layer_norm(x, weight, bias)``                       ln1 / ln2 of a block (model.py:45,51)
* ``causal_conv(x, weight, bias, ...)``                 the mixer's depthwise convolution + SiLU
* ``causal_conv_step(x, state, weight, bias)``          the same for one token per stream
* ``ssm_scan(x, dt, A, B, C, D, z, dt_bias, ...)``      the mixer's selective state space scan
* ``ssm_step(x, dt, state, A, B, C, D, z, dt_bias)``    the same for one token per stream

The sequence forms are differentiable in every floating argument (in reverse
mode and once: a backward pass with ``create_graph`` and inputs with a
forward-mode tangent are refused); the step forms update their state in place
and are for inference.  ``torch.jit.trace`` is refused too.

Sequences are ``[batch, length, channels]``.  Activations of one call share one
type (float32, bfloat16 or float16); their rows may be strided (a slice of a
wider projection needs no copy), other layouts are copied.  Parameters are
taken in float32 (other types are cast, and their gradients cast back); scan
states are float32, convolution windows have the activations' type.  ``lens``
(``[batch]``, int32 or int64, on the device) gives the valid length of each row:
what lies behind it is never read, and its outputs and gradients are zero.

All calls run on the tensors' device and torch's current stream, allocate
through torch, keep nothing, never synchronise, and can be captured into a CUDA
graph.  Equal inputs give equal bits, but unlike the codec's fused kernel these
operators do not promise a row the same bits in batches of different size.
There is no CPU path: tensors that are not on a CUDA device raise RuntimeError.
"""
from __future__ import annotations

import ctypes
import importlib

import torch  # noqa: F401  (before _boa_ops, which links to it)

from . import _native as _n

_ENTRY_POINTS = [n for n in _n.SIGNATURES if n.startswith(("boa_layer_norm", "boa_causal_conv", "boa_ssm_"))]


def _addresses():
    """The library's entry points for _boa_ops, on first use."""
    lib = _n.load()
    return {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in ["boa_last_error"] + _ENTRY_POINTS}


class _OnFirstUse:
    """Stands for _boa_ops until its first call, so that a program that runs only
    the codec does not load it; raises if it was not built."""

    def __getattr__(self, name):
        global _boa_ops
        try:
            module = importlib.import_module("._boa_ops", __package__)
        except ImportError as e:
            raise RuntimeError(f"_boa_ops is not built ({e}); run __graft_entry__.build()") from e
        module.bind(_addresses, _n.BoaError)
        _boa_ops = module
        return getattr(module, name)


_boa_ops = _OnFirstUse()


def layer_norm(x, weight, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (1 to 8192 wide); weight and bias are ``[width]``."""
    return _boa_ops.layer_norm(x, weight, bias, eps)


def causal_conv(x, weight, bias=None, *, silu: bool = True, state=None, lens=None, return_state: bool = False):
    """Depthwise causal convolution of ``x [batch, length, channels]`` with
    ``weight [channels, width]`` (or ``[channels, 1, width]``; width 2 to 4) and
    ``bias [channels]``, followed by SiLU unless ``silu`` is false.

    ``state [batch, width - 1, channels]`` holds the inputs before the first
    position, oldest first (zeros when None).  With ``return_state`` the result
    is ``(y, state behind each row's last valid position)``."""
    return _boa_ops.causal_conv(x, weight, bias, silu, state, lens, return_state)


def causal_conv_step(x, state, weight, bias=None, *, silu: bool = True):
    """One token of ``causal_conv`` for every stream: ``x [batch, channels]`` ->
    ``y [batch, channels]``; ``state [batch, width - 1, channels]`` (contiguous)
    moves on by one token in place."""
    return _boa_ops.causal_conv_step(x, state, weight, bias, silu)


def ssm_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, *, softplus: bool = True, state=None, lens=None,
             return_state: bool = False):
    """Selective state space scan over ``x, dt [batch, length, channels]``:

        d = softplus(dt + dt_bias)                      (dt + dt_bias when ``softplus`` is false)
        h_t = exp(d_t A) h_{t-1} + d_t x_t B_t          A [channels, 16], B, C [batch, length, 16]
        y_t = (C_t . h_t + D x_t) silu(z_t)             D [channels] and z [batch, length, channels] optional

    ``state [batch, channels, 16]`` (float32) is h before the first position
    (zeros when None).  With ``return_state`` the result is ``(y, h behind each
    row's last valid position)``."""
    return _boa_ops.ssm_scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, return_state)


def ssm_step(x, dt, state, A, B, C, D=None, z=None, dt_bias=None, *, softplus: bool = True):
    """One token of ``ssm_scan`` for every stream: ``x, dt, z [batch, channels]``,
    ``B, C [batch, 16]`` -> ``y [batch, channels]``; ``state [batch, channels, 16]``
    (float32, contiguous, 16-byte aligned) is updated in place."""
    return _boa_ops.ssm_step(x, dt, state, A, B, C, D, z, dt_bias, softplus)


def held_on_default_stream(parameters) -> bool:
    """Whether an autograd graph that is still alive would add to the gradient of
    one of ``parameters`` on the default stream: a backward pass must not be
    captured then."""
    return _boa_ops.held_on_default_stream(tuple(parameters))
