"""Drop-in for the reference ``model.py``: ``BoaConstrictor(d_model, num_layers,
vocab_size, device)`` returns a ``BoaBytePredictor`` with the reference's module
tree and state_dict keys (model.py:42-134, the key set that
portability_solved_cpp/convert_boa_weights.py:16-135 reads).

The Mamba mixer is this build's own module with mamba_ssm's parameter shapes
and initialisation recipe (mamba_ssm itself is not a dependency): d_state 16,
d_conv 4, expand 2, dt_rank ceil(d_model/16), in_proj/out_proj without bias,
dt_proj weight U(+-dt_rank^-0.5), dt_proj bias = softplus^-1 of a log-uniform
dt in [1e-3, 1e-1] floored at 1e-4, A_log = log(1..16), D = 1.

Inference (``init_stream`` / ``step`` / ``forward``) runs on the sm_100a kernel
in libboa_b200.so (``boa_model_step`` / ``boa_model_logits``) on a CUDA
device; there is no CPU execution path.

``forward_layers`` / ``step_layers`` run the same model layer by layer on the
module's own parameters (on the GPU, any d_model): the matrix products are
torch's, everything between them is ``boa_b200.ops``.  This is the path with
gradients, for prompts parallel over positions, and for ragged batches; its
probabilities agree with the fused kernel's to rounding, not bit for bit, so the
codec does not use it.
"""
from __future__ import annotations

import ctypes
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from boa_b200 import _native as _n
from boa_b200 import ops
from boa_b200.weights import flatten_state_dict

D_STATE = 16
D_CONV = 4
EXPAND = 2

# Projection operand formats of the kernel.  "tf32x3" (the default) splits every
# fp32 weight and activation into tf32 hi + lo halves whose products are summed
# in fp32: the arithmetic of the reference's fp32 nn.Linear to within fp32
# rounding.  "f16x2" carries the same 22 significant bits as an fp16 hi and an
# fp16 residual scaled by 2^11, at half the weight bytes, for activations
# below 65504 in magnitude (larger ones are reported, BOA_ERR_RANGE).  "tf32",
# "fp16" and "bf16" are faster, narrower alternatives ("bf16" is what the
# d_model-512 configuration specifies).
WEIGHT_FORMATS = {"tf32x3": _n.BOA_WEIGHTS_TF32X3, "f16x2": _n.BOA_WEIGHTS_F16X2, "tf32": _n.BOA_WEIGHTS_TF32,
                  "bf16": _n.BOA_WEIGHTS_BF16, "fp16": _n.BOA_WEIGHTS_F16}


def default_format(d_model: int) -> str:
    """The operand kind used when none is given: "f16x2" (fp32-equivalent; its
    probabilities at d_model 256 / 8 layers are within 1.5e-8 of an fp64
    evaluation, the reference's own fp32 arithmetic within 6e-9) for
    d_model <= 256, and "bf16" for d_model 512, where the split kinds do not
    fit shared memory and TMEM (the d_model-512 configuration specifies bf16)."""
    return "f16x2" if d_model <= 256 else "bf16"


class Mamba(nn.Module):
    """Parameters of one Mamba mixer (shapes and init as mamba_ssm.Mamba(d_model))."""

    def __init__(self, d_model: int, dt_min: float = 1e-3, dt_max: float = 1e-1, dt_init_floor: float = 1e-4):
        super().__init__()
        self.d_model = d_model
        self.d_state = D_STATE
        self.d_conv = D_CONV
        self.d_inner = EXPAND * d_model
        self.dt_rank = math.ceil(d_model / 16)
        E, R = self.d_inner, self.dt_rank
        self.in_proj = nn.Linear(d_model, 2 * E, bias=False)
        self.conv1d = nn.Conv1d(E, E, kernel_size=D_CONV, groups=E, padding=D_CONV - 1, bias=True)
        self.x_proj = nn.Linear(E, R + 2 * D_STATE, bias=False)
        self.dt_proj = nn.Linear(R, E, bias=True)
        std = R ** -0.5
        with torch.no_grad():
            nn.init.uniform_(self.dt_proj.weight, -std, std)
            dt = torch.exp(torch.rand(E) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
            dt = dt.clamp(min=dt_init_floor)
            self.dt_proj.bias.copy_(dt + torch.log(-torch.expm1(-dt)))
        A = torch.arange(1, D_STATE + 1, dtype=torch.float32).repeat(E, 1)
        self.A_log = nn.Parameter(torch.log(A))
        self.D = nn.Parameter(torch.ones(E))
        self.out_proj = nn.Linear(E, d_model, bias=False)

    def init_state(self, batch_size: int, device=None, dtype=None):
        """(convolution window [B, 3, E], scan state [B, E, 16] fp32) before the first token.  The window has
        the type of the activations: the weights' one, or that of the autocast region."""
        w = self.in_proj.weight
        device = torch.device(device) if device else w.device
        if dtype is None:
            dtype = torch.get_autocast_dtype(device.type) if torch.is_autocast_enabled(device.type) else w.dtype
        return (torch.zeros(batch_size, D_CONV - 1, self.d_inner, dtype=dtype, device=device),
                torch.zeros(batch_size, self.d_inner, D_STATE, dtype=torch.float32, device=device))

    def _split(self, dbc):
        return dbc.split([self.dt_rank, D_STATE, D_STATE], dim=-1)

    def forward(self, u, state=None, lens=None, return_state: bool = False):
        """u [B, L, d_model] -> [B, L, d_model], from ``state`` (zeros when None).
        ``lens`` [B] cuts each row; with ``return_state`` also the state behind
        every row's last valid position.  Differentiable."""
        conv, ssm = (None, None) if state is None else state
        x, z = self.in_proj(u).chunk(2, dim=-1)
        x, conv = ops.causal_conv(x, self.conv1d.weight, self.conv1d.bias, state=conv, lens=lens, return_state=True)
        dt, B, C = self._split(self.x_proj(x))
        dt = F.linear(dt, self.dt_proj.weight)
        y, ssm = ops.ssm_scan(x, dt, -torch.exp(self.A_log.float()), B, C, self.D, z, self.dt_proj.bias, state=ssm,
                              lens=lens, return_state=True)
        y = self.out_proj(y)
        return (y, (conv, ssm)) if return_state else y

    @torch.no_grad()
    def step(self, u, state):
        """One token of every stream: u [B, d_model] -> [B, d_model]; ``state``
        (from ``init_state`` or ``forward``) moves on in place."""
        conv, ssm = state
        x, z = self.in_proj(u).chunk(2, dim=-1)
        x = ops.causal_conv_step(x, conv, self.conv1d.weight, self.conv1d.bias)
        dt, B, C = self._split(self.x_proj(x))
        dt = F.linear(dt, self.dt_proj.weight)
        y = ops.ssm_step(x, dt, ssm, -torch.exp(self.A_log.float()), B, C, self.D, z, self.dt_proj.bias)
        return self.out_proj(y)


class MambaBlock(nn.Module):
    """ln1 -> mamba -> ln2 -> ff -> + x (model.py:42-65)."""

    def __init__(self, d_model: int):
        super().__init__()
        self.ln1 = nn.LayerNorm(d_model)
        self.mamba = Mamba(d_model)
        self.ln2 = nn.LayerNorm(d_model)
        self.ff = nn.Sequential(nn.Linear(d_model, 4 * d_model), nn.GELU(), nn.Linear(4 * d_model, d_model))

    def _finish(self, x, y):
        return x + self.ff(ops.layer_norm(y, self.ln2.weight, self.ln2.bias, self.ln2.eps))

    def forward(self, x, state=None, lens=None, return_state: bool = False):
        u = ops.layer_norm(x, self.ln1.weight, self.ln1.bias, self.ln1.eps)
        y, state = self.mamba(u, state, lens, return_state=True)
        y = self._finish(x, y)
        return (y, state) if return_state else y

    @torch.no_grad()
    def step(self, x, state):
        return self._finish(x, self.mamba.step(ops.layer_norm(x, self.ln1.weight, self.ln1.bias, self.ln1.eps), state))


class StreamState:
    """Per-stream recurrent state for ``step`` (replaces mamba_ssm's
    InferenceParams, model.py:104-106): conv windows + SSM states of every
    layer, resident on the device in the layout the kernel expects."""

    def __init__(self, model: "BoaBytePredictor", batch_size: int, device):
        self.batch_size = int(batch_size)
        self.device = torch.device(device)
        nb = model._native_handle(self.device).workspace_bytes(self.batch_size)
        self.workspace = torch.zeros(nb, dtype=torch.uint8, device=self.device)
        self.seqlen_offset = 0


class NativeModel:
    """Owns a boa_model handle built from a state_dict snapshot."""

    def __init__(self, sd, d_model: int, n_layers: int, vocab: int, weight_format: int, device_index: int):
        flat = flatten_state_dict(sd)
        h = ctypes.c_void_p()
        _n.call("boa_model_create", ctypes.byref(h), int(d_model), int(n_layers), int(vocab),
                flat.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(flat.size), int(weight_format),
                int(device_index))
        self.h = h
        self.device_index = device_index
        self.d_model, self.n_layers, self.vocab, self.weight_format = d_model, n_layers, vocab, weight_format

    def workspace_bytes(self, n: int) -> int:
        return int(_n.load().boa_model_workspace_bytes(self.h, int(n)))

    def set_time_block(self, positions: int) -> None:
        """Positions per kernel step for encode / logits runs: 0 (default: each
        launch chooses 4 or 8), 1, 4 or 8.  The output bits are the same."""
        _n.call("boa_model_set_time_block", self.h, int(positions))

    def time_block(self, n_chunks: int, positions: int) -> int:
        """Positions per kernel step an encode / logits launch of this shape takes."""
        tb = ctypes.c_int(0)
        _n.call("boa_model_time_block", self.h, int(n_chunks), int(positions), ctypes.byref(tb))
        return tb.value

    def check(self, stream=None) -> None:
        """Wait for `stream` (torch's current stream by default) and raise the
        device-side errors of this model's calls enqueued so far
        (boa_model_status: timeouts, overflowing streams, bad symbols)."""
        import torch
        if stream is None:
            stream = torch.cuda.current_stream(torch.device("cuda", self.device_index))
        _n.call("boa_model_status", self.h, ctypes.c_void_p(int(stream.cuda_stream)))

    def tile_bytes_per_step(self) -> int:
        v = ctypes.c_size_t()
        _n.call("boa_model_info", self.h, None, None, None, None, ctypes.byref(v))
        return int(v.value)

    def close(self):
        if getattr(self, "h", None) is not None and self.h.value:
            _n.load().boa_model_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class BoaBytePredictor(nn.Module):
    """Mamba model predicting the next byte (model.py:83-131)."""
    _captured = False       # whether a CUDA graph may hold a training step of these parameters

    def __init__(self, d_model=256, num_layers=4, vocab_size=256, weight_format: str | None = None):
        super().__init__()
        self.embedding = nn.Embedding(vocab_size, d_model)
        self.blocks = nn.ModuleList([MambaBlock(d_model) for _ in range(num_layers)])
        self.head = nn.Sequential(nn.Linear(d_model, d_model), nn.ReLU(), nn.Linear(d_model, vocab_size))
        self.d_model = d_model
        self.num_layers = num_layers
        self.vocab_size = vocab_size
        self.weight_format = weight_format or default_format(d_model)
        if self.weight_format not in WEIGHT_FORMATS:
            raise ValueError(f"unknown weight_format {weight_format!r}; one of {sorted(WEIGHT_FORMATS)}")
        self._native = {}

    # -- native handle management ---------------------------------------------
    def _param_key(self):
        return tuple((id(p), p._version) for p in self.parameters()), self.weight_format

    def _param_values(self):
        """All parameters in one tensor: what a replayed graph changes without moving a version."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured training step may have changed the parameters, and they cannot be read "
                               "while another capture runs: capture the fused kernel with a model of its own")
        return torch.cat([p.detach().reshape(-1).float() for p in self.parameters()])

    def _native_handle(self, device) -> NativeModel:
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("boa_b200 inference runs on CUDA devices only (no CPU path)")
        _n.require_cuda()
        idx = device.index if device.index is not None else torch.cuda.current_device()
        key = (idx,) + self._param_key()
        nm = self._native.get(idx)
        values = self._param_values() if self._captured else None
        if nm is None or nm[0] != key or (values is not None and (nm[2] is None or not torch.equal(nm[2], values))):
            sd = {k: v.detach().float().cpu() for k, v in self.state_dict().items()}
            self._native[idx] = (key, NativeModel(sd, self.d_model, self.num_layers, self.vocab_size,
                                                  WEIGHT_FORMATS[self.weight_format], idx), values)
        return self._native[idx][1]

    def native(self, device=None) -> NativeModel:
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        return self._native_handle(device)

    # -- reference API ----------------------------------------------------------
    @torch.inference_mode()
    def init_stream(self, max_len: int, batch_size: int = 1, device=None, dtype=None):
        if device is None:
            device = "cuda"
        return StreamState(self, batch_size, device)

    @torch.inference_mode()
    def step(self, byte_t: torch.LongTensor, inf: StreamState) -> torch.Tensor:
        """byte_t [B] -> logits [B, vocab] (model.py:108-117)."""
        dev = inf.device
        nm = self._native_handle(dev)
        toks = byte_t.reshape(-1).to(device=dev, dtype=torch.int32).contiguous()
        B = toks.numel()
        if B != inf.batch_size:
            raise ValueError(f"step got {B} tokens for a stream of batch {inf.batch_size}")
        out = torch.empty((B, self.vocab_size), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            _n.call("boa_model_step", nm.h, B, ctypes.c_void_p(toks.data_ptr()), ctypes.c_void_p(out.data_ptr()),
                    ctypes.c_void_p(inf.workspace.data_ptr()), ctypes.c_size_t(inf.workspace.numel()),
                    ctypes.c_void_p(_n.stream_ptr(dev)))
        inf.seqlen_offset += 1
        return out

    @torch.inference_mode()
    def forward(self, x, inference_params=None):
        """x [B, L] -> logits [B, L, vocab] from a zero state (model.py:97-101)."""
        dev = x.device if x.is_cuda else torch.device("cuda", torch.cuda.current_device())
        nm = self._native_handle(dev)
        B, L = x.shape
        toks = x.to(device=dev, dtype=torch.int32).contiguous()
        out = torch.empty((B, L, self.vocab_size), dtype=torch.float32, device=dev)
        ws = torch.empty(nm.workspace_bytes(B), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _n.call("boa_model_logits", nm.h, B, L, ctypes.c_void_p(toks.data_ptr()),
                    ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(ws.data_ptr()),
                    ctypes.c_size_t(ws.numel()), ctypes.c_void_p(_n.stream_ptr(dev)))
        return out


    # -- layer by layer on the module's own parameters ---------------------------
    def _check_tokens(self, who, x, dims):
        if x.dim() != dims:
            raise ValueError(f"{who}: tokens must be {'[batch, length]' if dims == 2 else '[batch]'}, "
                             f"got {tuple(x.shape)}")
        if not self.embedding.weight.is_cuda:
            raise RuntimeError(f"{who} runs on CUDA devices only (no CPU path): move the model with .cuda()")

    def _check_state(self, who, state):
        if len(state) != len(self.blocks):
            raise ValueError(f"{who}: the model has {len(self.blocks)} blocks, the state holds {len(state)}")

    def _embed(self, x, lens=None):
        """Embedded tokens; what a row holds behind its valid length is no token (padding of any value)."""
        x = x.to(self.embedding.weight.device).long()
        if lens is not None:
            if lens.shape != x.shape[:1]:
                raise ValueError(f"lens must have shape {tuple(x.shape[:1])}, got {tuple(lens.shape)}")
            x = x.masked_fill(torch.arange(x.shape[1], device=x.device) >= lens[:, None], 0)
        return self.embedding(x)

    def forward_layers(self, x, state=None, lens=None, return_state: bool = False):
        """x [B, L] -> logits [B, L, vocab], differentiable in every parameter.

        ``lens`` [B] gives the valid length of each row (what x holds behind it
        is not read, the logits there mean nothing).  ``state`` continues a
        sequence; with ``return_state`` the result is (logits, state behind
        every row's last valid position) for a later call or ``step_layers``."""
        self._check_tokens("forward_layers", x, 2)
        if state is not None:
            self._check_state("forward_layers", state)
        self._captured |= torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing()
        h = self._embed(x, lens)
        out = []
        for i, block in enumerate(self.blocks):
            h, s = block(h, None if state is None else state[i], lens, return_state=True)
            out.append(s)
        logits = self.head(h)
        return (logits, out) if return_state else logits

    def init_layers(self, batch_size: int, dtype=None):
        """The state before the first byte, for ``step_layers``."""
        return [b.mamba.init_state(batch_size, dtype=dtype) for b in self.blocks]

    @torch.no_grad()
    def step_layers(self, byte_t, state):
        """byte_t [B] -> logits [B, vocab]; ``state`` moves on in place."""
        self._check_tokens("step_layers", byte_t, 1)
        self._check_state("step_layers", state)
        h = self.embedding(byte_t.to(self.embedding.weight.device).long())
        for block, s in zip(self.blocks, state):
            h = block.step(h, s)
        return self.head(h)


def BoaConstrictor(d_model=256, num_layers=4, vocab_size=256, device="cuda", weight_format: str | None = None):
    """Construct a BoaBytePredictor (model.py:5-134).  Parameters are created on
    the CPU with the module-construction order of the reference (embedding,
    blocks, head) so a given torch seed always yields the same weights; the
    codec moves nothing to the GPU but the packed kernel weights."""
    model = BoaBytePredictor(d_model=d_model, num_layers=num_layers, vocab_size=vocab_size,
                             weight_format=weight_format)
    i = 0
    for m in model.modules():
        if isinstance(m, Mamba):
            m.layer_idx = i
            i += 1
    return model


def seeded_model(d_model: int, num_layers: int, vocab_size: int = 256, seed: int = 0,
                 weight_format: str | None = None) -> BoaBytePredictor:
    """The benchmark/test model: torch.manual_seed(seed) then construction."""
    torch.manual_seed(seed)
    return BoaConstrictor(d_model=d_model, num_layers=num_layers, vocab_size=vocab_size, device="cpu",
                          weight_format=weight_format)
