"""Training-side evaluation (train.py:9-22): bits per byte of a model over a
loader of byte sequences, through the model's forward pass.

BoaBytePredictor.forward runs the fused sm_100a kernel in logits mode with
time blocks of 4 positions (the same kernel and weight tiles as compression),
so evaluation costs one launch per batch instead of one per byte.

``train_step`` is one optimizer step on the layer-by-layer path
(``BoaBytePredictor.forward_layers``), whose operators have backward kernels.
The reference's training program around it (train.py:24 onwards: mixed
precision, checkpoints every epoch) is out of scope for this build and raises.
"""
from __future__ import annotations

import math

import torch

from boa_b200 import ops


@torch.inference_mode()
def evaluate_bpp(model, loader, criterion, device="cuda", vocab_size=256) -> float:
    """Mean next-byte negative log-likelihood over every position of every
    batch, in bits: each batch [B, L] predicts bytes 1..L-1 from 0..L-2."""
    model.eval()
    nll_sum = 0.0
    count = 0
    for batch in loader:
        inputs = batch[:, :-1].to(device)
        targets = batch[:, 1:].to(device)
        logits = model(inputs)                             # [B, L-1, vocab]
        loss = criterion(logits.reshape(-1, vocab_size), targets.reshape(-1).long())
        nll_sum += float(loss.item()) * targets.numel()
        count += targets.numel()
    return nll_sum / max(count, 1) / math.log(2.0)


def train_step(model, batch, optimizer, criterion, lens=None) -> torch.Tensor:
    """One step on a batch of byte rows [B, L]: predict bytes 1..L-1 from
    0..L-2, ``criterion(logits, targets)``, backward, ``optimizer.step()``.
    ``lens`` [B] is the number of valid bytes of each row; what lies behind
    takes no part.  Returns the loss (on the device, nothing is synchronised).

    Called within ``torch.autocast``, the forward part and the loss run in it,
    the backward pass and the optimizer outside of it; the casts of the weights
    that autocast keeps for its region are dropped, since the step changes them.

    It can be captured into a CUDA graph, behind a few steps on another stream.
    Autograd adds to a parameter's gradient on the stream of the oldest graph
    that is alive; on the default stream the capture would end the process, so
    it is refused while an output of an earlier call keeps such a graph."""
    dev = model.embedding.weight.device
    if dev.type == "cuda" and torch.cuda.is_current_stream_capturing() and ops.held_on_default_stream(model.parameters()):
        raise RuntimeError("train_step cannot be captured while a loss or an output of an earlier call keeps its autograd "
                           "graph alive: delete it first")
    batch = batch.to(dev)
    inputs, targets = batch[:, :-1], batch[:, 1:].long()
    if lens is not None:
        lens = (lens.to(dev) - 1).clamp(min=0)
        live = torch.arange(targets.shape[1], device=dev)[None, :] < lens[:, None]
        targets = torch.where(live, targets, torch.full_like(targets, -100))     # cross_entropy's ignore_index
    optimizer.zero_grad(set_to_none=True)
    logits = model.forward_layers(inputs, lens=lens)
    loss = criterion(logits.reshape(-1, logits.shape[-1]), targets.reshape(-1))
    with torch.autocast(dev.type, enabled=False):
        loss.backward()
        optimizer.step()
    torch.clear_autocast_cache()
    return loss.detach()


def train(*args, **kwargs):
    raise NotImplementedError("training (train.py:24-) is not part of the compress/decompress hot path; "
                              "train with the reference code and load the state_dict here")
