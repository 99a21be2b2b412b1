"""Dropout masks for training steps replayed from HIP graphs.

The dropout kernels (attention weights, layer norm + dropout) decide every element by a hash of its
position and the call's two seeds.  The seeds are by-value kernel arguments: a captured graph freezes
them, and a replayed step would draw the same masks for ever, where the reference draws fresh ones at
every call (nn.Dropout, src/models/lmu_encoder.py:45, 86, 232).  The library therefore adds a 32-bit
counter read from DEVICE memory to the seeds when the kernels run (C ABI lmufft_dropout_epoch); the
captured step increments the counter as its first node, so every replay sees a new value, and the
forward and backward kernels of one step see the same one.

dropout_add is the dropout that stands alone, with the residual it is added to (HIP kernel k_dropout_add).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

_EPOCHS = {}  # device index -> int32 tensor [1], registered with the library for that device


def _index(device) -> int:
    device = torch.device(device)
    return device.index if device.index is not None else torch.cuda.current_device()


def dropout_epoch(device) -> torch.Tensor:
    """The device's epoch counter, created and registered with the library on first use.  Must first be
    called outside a graph capture (its allocation and zero-fill must not become graph nodes)."""
    idx = _index(device)
    t = _EPOCHS.get(idx)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("asr_amd: a dropout step is being captured into a HIP graph before the device's dropout "
                               "epoch counter exists; call asr_amd.dropout.dropout_epoch(device) before the capture "
                               "(GradBuckets.capture_* do) and increment it inside the captured step (bump_dropout_epoch)")
        dev = torch.device("cuda", idx)
        t = torch.zeros(1, dtype=torch.int32, device=dev)
        with torch.cuda.device(dev):
            _lib.check(_lib.lib.lmufft_dropout_epoch(ctypes.c_void_p(t.data_ptr())), "lmufft_dropout_epoch")
        _EPOCHS[idx] = t
    return t


def epoch_registered(device) -> bool:
    return _index(device) in _EPOCHS


def bump_dropout_epoch(device) -> None:
    """Increment the device's counter on the current stream (inside a capture: a node of the graph)."""
    dropout_epoch(device).add_(1)


def check_capturable(device, p_drop: float, seeds_given: bool) -> None:
    """Raises when a dropout call with default seeds is being captured and no epoch counter is registered:
    the replayed step would reuse one mask for ever."""
    if p_drop > 0 and not seeds_given and torch.cuda.is_current_stream_capturing() and not epoch_registered(device):
        dropout_epoch(device)  # raises with the explanation


_dropout_calls = 0
_ops = None  # the bound operators, loaded by the first dropout_add: what else is here needs the C library only


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, p_drop: float = 0.1, seeds=None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """residual + dropout(x) with autograd, one pass in each direction and no stored mask: an element of x [..., C] is
    kept with probability 1 - p_drop, scaled by 1 / (1 - p_drop), and decided by its row, its column and the call's seeds.

    x, residual: float32 or bfloat16 each, of one shape; the result has `out_dtype`, by default the promoted dtype.
    `seeds` = (seed0, seed1), two 32-bit integers that name the mask; by default torch's seed and a per-process call
    counter.  Under HIP graph capture the seeds are frozen and the device's epoch counter gives every replay its own mask
    (see above); without that counter such a capture raises."""
    global _dropout_calls, _ops
    if _ops is None:
        from ._call import ops as _ops
    if not 0.0 <= p_drop < 1.0:
        raise ValueError(f"dropout probability has to be in [0, 1), got {p_drop}")
    if seeds is None:
        if x.is_cuda:
            check_capturable(x.device, p_drop, False)
        if p_drop > 0:
            _dropout_calls += 1
        seeds = (torch.initial_seed() & 0xFFFFFFFF, 0x44520000 ^ (_dropout_calls & 0xFFFFFFFF))
    return _ops.dropout_add(x, residual, p_drop, int(seeds[0]) & 0xFFFFFFFF, int(seeds[1]) & 0xFFFFFFFF, out_dtype)
