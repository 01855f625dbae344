"""Operators of a Mamba block outside its matrix products, on the sm_100a
kernels of libboa_b200.so (``boa_layer_norm``, ``boa_causal_conv``,
``boa_ssm_scan`` and their backward and one-token forms):

* ``layer_norm(x, weight, bias)``                       ln1 / ln2 of a block (model.py:45,51)
* ``causal_conv(x, weight, bias, ...)``                 the mixer's depthwise convolution + SiLU
* ``causal_conv_step(x, state, weight, bias)``          the same for one token per stream
* ``ssm_scan(x, dt, A, B, C, D, z, dt_bias, ...)``      the mixer's selective state space scan
* ``ssm_step(x, dt, state, A, B, C, D, z, dt_bias)``    the same for one token per stream

The sequence forms are differentiable in every floating argument (once; there
is no second derivative); the step forms update their state in place and are
for inference.

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

import torch
from torch.autograd.function import once_differentiable

from . import _native as _n

D_STATE = 16

_DTYPES = {torch.float32: _n.BOA_DTYPE_F32, torch.bfloat16: _n.BOA_DTYPE_BF16, torch.float16: _n.BOA_DTYPE_F16}


# ------------------------------------------------------------------ arguments
# The host side of a one-token call is most of its time, so the checks compare
# shapes and device indexes directly and the library's functions are looked up once.
def _kind(who, x):
    k = _DTYPES.get(x.dtype)
    if k is None:
        raise ValueError(f"{who}: x must be float32, bfloat16 or float16, not {x.dtype}")
    return k


def _shape(who, name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{who}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _same(who, x, name, t):
    """Activations of one call share x's type."""
    if t.dtype != x.dtype:
        raise ValueError(f"{who}: {name} must have the type of x ({x.dtype}), got {t.dtype}")


def _on_device(who, x, *others):
    """The index of the CUDA device that holds every tensor."""
    index = x.get_device()
    if index < 0:
        raise RuntimeError(f"{who} runs on CUDA devices only (no CPU path)")
    for t in others:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"{who}: all tensors must be on {x.device}, got one on {t.device}")
    return index


def _param(t):
    """A parameter as contiguous, 16-byte aligned fp32 (differentiable cast)."""
    if t is None:
        return None
    if t.dtype != torch.float32:
        t = t.float()
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t):
    """Channels contiguous; other strides stay as they are."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _lens(who, lens, batch, length):
    if lens is None:
        return None
    if lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{who}: lens must be int32 or int64, not {lens.dtype}")
    _shape(who, "lens", lens, (batch,))
    if lens.dtype == torch.int64:
        lens = lens.clamp(0, length).to(torch.int32)
    return lens.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


_functions = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _n.stream_ptr)   # handle of the device's current stream


def _fn(name):
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(_n.load(), name)
    return f


def _call(name, index, *args):
    """One library call on device `index`'s current stream."""
    f = _functions.get(name) or _fn(name)
    if torch.cuda.current_device() == index:
        rc = f(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index))
    if rc:
        _n.check(rc, name)


def _workspace(nbytes, like):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ----------------------------------------------------------------- layer norm
def _norm_forward(x, weight, bias, eps, keep_stats):
    rows, width = x.shape
    y = x.new_empty((rows, width))
    stats = x.new_empty((rows, 2), dtype=torch.float32) if keep_stats else None
    index = x.get_device()
    _call("boa_layer_norm", index, rows, width, _DTYPES[x.dtype], x.data_ptr(), x.stride(0), weight.data_ptr(),
          _ptr(bias), eps, y.data_ptr(), _ptr(stats), index)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.with_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        rows, width = x.shape
        dy = _rows(dy)
        dx = x.new_empty((rows, width))
        dw = torch.empty_like(weight)
        db = torch.empty_like(weight) if ctx.with_bias else None
        kind, index = _DTYPES[x.dtype], x.get_device()
        nbytes = _fn("boa_layer_norm_workspace_bytes")(rows, width, kind)
        ws = _workspace(nbytes, x)
        _call("boa_layer_norm_backward", index, rows, width, kind, x.data_ptr(), x.stride(0), dy.data_ptr(),
              dy.stride(0), weight.data_ptr(), stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(ws),
              nbytes, index)
        return dx, dw, db, None


def layer_norm(x, weight, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (1 to 8192 wide); weight and bias are ``[width]``."""
    who = "layer_norm"
    _kind(who, x)
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{who}: x needs a last axis of at least one element, got shape {tuple(shape)}")
    width = shape[-1]
    _shape(who, "weight", weight, (width,))
    if bias is not None:
        _shape(who, "bias", bias, (width,))
    _on_device(who, x, weight, bias)
    weight, bias = _param(weight), _param(bias)
    flat = _rows(x if len(shape) == 2 else x.reshape(-1, width))
    if _wants_grad(x, weight, bias):
        y = _LayerNorm.apply(flat, weight, bias, float(eps))
    else:
        y, _ = _norm_forward(flat, weight, bias, float(eps), False)
    return y if len(shape) == 2 else y.view(shape)


# --------------------------------------------------------- causal convolution
def _conv_args(x, weight, bias, silu, state, lens, y=None, state_out=None):
    shape, strides = x.shape, x.stride()
    step = len(shape) == 2
    return _n.ConvArgs(_DTYPES[x.dtype], shape[0], 0 if step else shape[1], shape[-1], weight.shape[1], int(silu),
                       x.get_device(), 0, x.data_ptr(), strides[0], 0 if step else strides[1], weight.data_ptr(),
                       _ptr(bias), _ptr(state), _ptr(lens), _ptr(y), _ptr(state_out))


def _conv_forward(x, weight, bias, silu, state, lens, return_state):
    b, length, e = x.shape
    y = x.new_empty((b, length, e))
    out = x.new_empty((b, weight.shape[1] - 1, e)) if return_state else None
    a = _conv_args(x, weight, bias, silu, state, lens, y, out)
    _call("boa_causal_conv", a.device, ctypes.byref(a))
    return y, out


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lens, silu, return_state):
        ctx.set_materialize_grads(False)
        y, out = _conv_forward(x, weight, bias, silu, state, lens, return_state)
        ctx.save_for_backward(x, weight, bias, state, lens)
        ctx.silu = silu
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        x, weight, bias, state, lens = ctx.saved_tensors
        a = _conv_args(x, weight, bias, ctx.silu, state, lens)
        dy = x.new_zeros(x.shape) if dy is None else _rows(dy)
        dout = None if dout is None else dout.contiguous()
        dx = x.new_empty(x.shape)
        dw = torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        ds = None if state is None else torch.empty_like(state)
        a.dy, a.dy_bs, a.dy_ts, a.dstate_out = _ptr(dy), dy.stride(0), dy.stride(1), _ptr(dout)
        a.dx, a.dweight, a.dbias, a.dstate = _ptr(dx), _ptr(dw), _ptr(db), _ptr(ds)
        a.workspace_bytes = _fn("boa_causal_conv_workspace_bytes")(ctypes.byref(a))
        ws = _workspace(a.workspace_bytes, x)
        a.workspace = _ptr(ws)
        _call("boa_causal_conv_backward", a.device, ctypes.byref(a))
        return dx, dw, db, ds, None, None, None


def _conv_weight(who, weight, channels):
    if weight.dim() == 3 and weight.shape[1] == 1:      # nn.Conv1d(groups=channels).weight
        weight = weight[:, 0]
    if weight.dim() != 2 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"{who}: weight must be [{channels}, width] or [{channels}, 1, width] with width 2, 3 or 4, "
                         f"got {tuple(weight.shape)}")
    return weight


def causal_conv(x, weight, bias=None, *, silu: bool = True, state=None, lens=None, return_state: bool = False):
    """Depthwise causal convolution of ``x [batch, length, channels]`` with
    ``weight [channels, width]`` (or ``[channels, 1, width]``; width 2 to 4) and
    ``bias [channels]``, followed by SiLU unless ``silu`` is false.

    ``state [batch, width - 1, channels]`` holds the inputs before the first
    position, oldest first (zeros when None).  With ``return_state`` the result
    is ``(y, state behind each row's last valid position)``."""
    who = "causal_conv"
    _kind(who, x)
    if x.dim() != 3 or x.shape[2] < 1:
        raise ValueError(f"{who}: x must be [batch, length, channels], got {tuple(x.shape)}")
    b, length, e = x.shape
    weight = _conv_weight(who, weight, e)
    if bias is not None:
        _shape(who, "bias", bias, (e,))
    if state is not None:
        _shape(who, "state", state, (b, weight.shape[1] - 1, e))
        _same(who, x, "state", state)
    lens = _lens(who, lens, b, length)
    _on_device(who, x, weight, bias, state, lens)
    weight, bias, x = _param(weight), _param(bias), _rows(x)
    state = None if state is None else state.contiguous()
    if _wants_grad(x, weight, bias, state):
        y, out = _CausalConv.apply(x, weight, bias, state, lens, silu, return_state)
    else:
        y, out = _conv_forward(x, weight, bias, silu, state, lens, return_state)
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, silu: bool = True):
    """One token of ``causal_conv`` for every stream: ``x [batch, channels]`` ->
    ``y [batch, channels]``; ``state [batch, width - 1, channels]`` (contiguous)
    moves on by one token in place."""
    who = "causal_conv_step"
    _kind(who, x)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{who}: x must be [batch, channels], got {tuple(x.shape)}")
    weight = _conv_weight(who, weight, x.shape[1])
    if bias is not None:
        _shape(who, "bias", bias, (x.shape[1],))
    _shape(who, "state", state, (x.shape[0], weight.shape[1] - 1, x.shape[1]))
    _same(who, x, "state", state)
    if not state.is_contiguous():
        raise ValueError(f"{who}: state is updated in place and must be contiguous")
    _on_device(who, x, state, weight, bias)
    if _wants_grad(x, state, weight, bias):
        raise RuntimeError(f"{who} has no gradient: call it under torch.no_grad(), or use causal_conv")
    weight, bias, x = _param(weight), _param(bias), _rows(x)
    y = x.new_empty(x.shape)
    a = _conv_args(x, weight, bias, silu, None, None, y, state)
    _call("boa_causal_conv_step", a.device, ctypes.byref(a))
    return y


# ----------------------------------------------------- selective state space scan
def _ssm_args(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, y=None, state_out=None, checkpoints=None):
    shape = x.shape
    if len(shape) == 2:
        length, xs, ds, Bs, Cs = 0, (x.stride(0), 0), (dt.stride(0), 0), (B.stride(0), 0), (C.stride(0), 0)
        zs = (0, 0) if z is None else (z.stride(0), 0)
    else:
        length, xs, ds, Bs, Cs = shape[1], x.stride(), dt.stride(), B.stride(), C.stride()
        zs = (0, 0) if z is None else z.stride()
    return _n.SsmArgs(_DTYPES[x.dtype], shape[0], length, shape[-1], D_STATE, int(softplus), x.get_device(), 0,
                      x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(),
                      xs[0], xs[1], ds[0], ds[1], zs[0], zs[1], Bs[0], Bs[1], Cs[0], Cs[1],
                      A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state), _ptr(lens), _ptr(y), _ptr(state_out),
                      _ptr(checkpoints))


def _ssm_forward(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, return_state, keep):
    b, length, e = x.shape
    y = x.new_empty((b, length, e))
    out = A.new_empty((b, e, D_STATE)) if return_state else None
    a = _ssm_args(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, y, out)
    r = ctypes.byref(a)
    checkpoints = _workspace(_fn("boa_ssm_checkpoint_bytes")(r), x) if keep else None
    a.checkpoints = _ptr(checkpoints)
    a.workspace_bytes = _fn("boa_ssm_workspace_bytes")(r, 0)
    ws = _workspace(a.workspace_bytes, x)
    a.workspace = _ptr(ws)
    _call("boa_ssm_scan", a.device, r)
    return y, out, checkpoints


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, lens, softplus, return_state):
        ctx.set_materialize_grads(False)
        y, out, checkpoints = _ssm_forward(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, return_state, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, state, lens, checkpoints)
        ctx.softplus = softplus
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        x, dt, A, B, C, D, z, dt_bias, state, lens, checkpoints = ctx.saved_tensors
        a = _ssm_args(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, state, lens, checkpoints=checkpoints)
        dy = x.new_zeros(x.shape) if dy is None else _rows(dy)
        dout = None if dout is None else dout.contiguous()
        fresh = lambda t: None if t is None else t.new_empty(t.shape)  # noqa: E731
        dx, ddt, dA, dB, dC, dD, dz, dbias, ds = (fresh(t) for t in (x, dt, A, B, C, D, z, dt_bias, state))
        a.dy, a.dy_bs, a.dy_ts, a.dstate_out = _ptr(dy), dy.stride(0), dy.stride(1), _ptr(dout)
        a.dx, a.ddt, a.dA, a.dB, a.dC = _ptr(dx), _ptr(ddt), _ptr(dA), _ptr(dB), _ptr(dC)
        a.dD, a.dz, a.ddt_bias, a.dstate = _ptr(dD), _ptr(dz), _ptr(dbias), _ptr(ds)
        r = ctypes.byref(a)
        a.workspace_bytes = _fn("boa_ssm_workspace_bytes")(r, 1)
        ws = _workspace(a.workspace_bytes, x)
        a.workspace = _ptr(ws)
        _call("boa_ssm_scan_backward", a.device, r)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, ds, None, None, None


def _ssm_check(who, x, dt, A, B, C, D, z, dt_bias, dims):
    _kind(who, x)
    shape = x.shape
    if len(shape) != dims or shape[-1] < 1:
        raise ValueError(f"{who}: x must be [batch, {'length, ' if dims == 3 else ''}channels], got {tuple(shape)}")
    e, bc = shape[-1], (*shape[:-1], D_STATE)
    _shape(who, "dt", dt, shape)
    _shape(who, "A", A, (e, D_STATE))
    _shape(who, "B", B, bc)
    _shape(who, "C", C, bc)
    if D is not None:
        _shape(who, "D", D, (e,))
    if dt_bias is not None:
        _shape(who, "dt_bias", dt_bias, (e,))
    if z is not None:
        _shape(who, "z", z, shape)
        _same(who, x, "z", z)
    _same(who, x, "dt", dt)
    _same(who, x, "B", B)
    _same(who, x, "C", C)


def _state32(who, state, x):
    _shape(who, "state", state, (x.shape[0], x.shape[-1], D_STATE))
    if state.dtype != torch.float32:
        raise ValueError(f"{who}: state must be float32, not {state.dtype}")


def ssm_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, *, softplus: bool = True, state=None, lens=None,
             return_state: bool = False):
    """Selective state space scan over ``x, dt [batch, length, channels]``:

        d = softplus(dt + dt_bias)                      (dt + dt_bias when ``softplus`` is false)
        h_t = exp(d_t A) h_{t-1} + d_t x_t B_t          A [channels, 16], B, C [batch, length, 16]
        y_t = (C_t . h_t + D x_t) silu(z_t)             D [channels] and z [batch, length, channels] optional

    ``state [batch, channels, 16]`` (float32) is h before the first position
    (zeros when None).  With ``return_state`` the result is ``(y, h behind each
    row's last valid position)``."""
    who = "ssm_scan"
    _ssm_check(who, x, dt, A, B, C, D, z, dt_bias, 3)
    if state is not None:
        _state32(who, state, x)
    lens = _lens(who, lens, x.shape[0], x.shape[1])
    _on_device(who, x, dt, A, B, C, D, z, dt_bias, state, lens)
    A, D, dt_bias, state = _param(A), _param(D), _param(dt_bias), _param(state)
    x, dt, B, C, z = _rows(x), _rows(dt), _rows(B), _rows(C), _rows(z)
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, state):
        y, out = _SsmScan.apply(x, dt, A, B, C, D, z, dt_bias, state, lens, softplus, return_state)
    else:
        y, out, _ = _ssm_forward(x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, return_state, False)
    return (y, out) if return_state else y


def ssm_step(x, dt, state, A, B, C, D=None, z=None, dt_bias=None, *, softplus: bool = True):
    """One token of ``ssm_scan`` for every stream: ``x, dt, z [batch, channels]``,
    ``B, C [batch, 16]`` -> ``y [batch, channels]``; ``state [batch, channels, 16]``
    (float32, contiguous, 16-byte aligned) is updated in place."""
    who = "ssm_step"
    _ssm_check(who, x, dt, A, B, C, D, z, dt_bias, 2)
    _state32(who, state, x)
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"{who}: state is updated in place and must be contiguous and 16-byte aligned")
    _on_device(who, x, dt, state, A, B, C, D, z, dt_bias)
    if _wants_grad(x, dt, state, A, B, C, D, z, dt_bias):
        raise RuntimeError(f"{who} has no gradient: call it under torch.no_grad(), or use ssm_scan")
    A, D, dt_bias = _param(A), _param(D), _param(dt_bias)
    x, dt, B, C, z = _rows(x), _rows(dt), _rows(B), _rows(C), _rows(z)
    y = x.new_empty(x.shape)
    a = _ssm_args(x, dt, A, B, C, D, z, dt_bias, softplus, None, None, y, state)
    _call("boa_ssm_step", a.device, ctypes.byref(a))
    return y
