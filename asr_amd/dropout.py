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
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import dense, on_device

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


_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_dropout_calls = 0


def _run(x, residual, p_drop, seed0, seed1, out_dtype):
    """residual + dropout(x), both dense; one pass."""
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    C = x.shape[-1]
    with on_device(x.device) as stream:
        rc = _lib.lib.lmufft_dropout_add(
            x.data_ptr(), _DTYPES[x.dtype], None if residual is None else residual.data_ptr(),
            0 if residual is None else _DTYPES[residual.dtype], x.numel() // C, C, p_drop, seed0, seed1, out.data_ptr(),
            _DTYPES[out_dtype], stream)
    if rc:
        _lib.check(rc, "lmufft_dropout_add")
    return out


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p_drop, seed0, seed1, out_dtype):
        ctx.conf = (p_drop, seed0, seed1, x.dtype, None if residual is None else residual.dtype)
        return _run(dense(x), None if residual is None else dense(residual), p_drop, seed0, seed1, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p_drop, seed0, seed1, x_dtype, res_dtype = ctx.conf
        dx = dres = None
        if ctx.needs_input_grad[0]:
            d = dy if dy.dtype in _DTYPES else dy.float()
            dx = _run(dense(d), None, p_drop, seed0, seed1, x_dtype)
        if ctx.needs_input_grad[1]:
            dres = dy.to(res_dtype)
        return dx, dres, None, None, None, None


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor] = None, p_drop: float = 0.1, seeds=None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """residual + dropout(x) with autograd, one pass in each direction and no stored mask: an element of x [..., C] is
    kept with probability 1 - p_drop, scaled by 1 / (1 - p_drop), and decided by its row, its column and the call's seeds.

    x, residual: float32 or bfloat16 each, of one shape; the result has `out_dtype`, by default the promoted dtype.
    `seeds` = (seed0, seed1), two 32-bit integers that name the mask; by default torch's seed and a per-process call
    counter.  Under HIP graph capture the seeds are frozen and the device's epoch counter gives every replay its own mask
    (see above); without that counter such a capture raises."""
    global _dropout_calls
    for name, t in (("x", x), ("residual", residual)):
        if t is None:
            continue
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"dropout_add: `{name}` is {t.dtype}; supported dtypes are float32 and bfloat16")
        if not t.is_cuda:
            raise RuntimeError(f"dropout_add: `{name}` lives on {t.device}; the kernel runs only on a GPU "
                               "(there is no CPU fallback)")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"dropout_add: x must be [..., channels], got {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise RuntimeError(f"dropout_add: residual {tuple(residual.shape)} on {residual.device} does not match x "
                           f"{tuple(x.shape)} on {x.device}")
    if not 0.0 <= p_drop < 1.0:
        raise ValueError(f"dropout probability has to be in [0, 1), got {p_drop}")
    if out_dtype is None:
        out_dtype = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
    if out_dtype not in _DTYPES:
        raise RuntimeError(f"dropout_add: output dtype {out_dtype} is not supported")
    check_capturable(x.device, p_drop, seeds is not None)
    if seeds is None:
        if p_drop > 0:
            _dropout_calls += 1
        seeds = (torch.initial_seed() & 0xFFFFFFFF, 0x44520000 ^ (_dropout_calls & 0xFFFFFFFF))
    return _DropoutAdd.apply(x, residual, float(p_drop), int(seeds[0]) & 0xFFFFFFFF, int(seeds[1]) & 0xFFFFFFFF, out_dtype)
