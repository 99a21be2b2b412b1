"""Group norm with an activation, channels last, on the GPU (HIP kernels k_gn_rows, k_gn_stats, k_gn_apply and their
backwards).

    y = act((x - mean) / sqrt(var + eps) * weight + bias)

x [B, T, C]: one mean and (biased) variance for each utterance and group of C / num_groups neighbouring channels, over the
frames inside its length; frames behind it are not read, their outputs and gradients are zeros.  x [N, C]: every row is a
sample of its own -- with num_groups = heads, the norm of each frame's heads behind an attention.  Beside the layer norm of
asr_amd/layernorm.py, which has one group, one sample a row, and no activation.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import dense, frames_of, on_device, ptr
from .parallel import adopt, grad_slot, run_deferred_sums

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2}
MAX_WIDTH = 1024


def _check(what, x, num_groups, weight, bias, activation, out_dtype):
    if x.dtype not in _DTYPES or out_dtype not in _DTYPES:
        raise RuntimeError(f"{what}: supported dtypes are float32 and bfloat16, got {x.dtype} and an output of {out_dtype}")
    if x.dim() not in (2, 3):
        raise RuntimeError(f"{what}: x must be [batch, frames, channels] or [rows, channels], got {tuple(x.shape)}")
    C = x.shape[-1]
    if num_groups <= 0 or C == 0 or C % num_groups:
        raise RuntimeError(f"{what}: {C} channels do not split into {num_groups} groups")
    if C > MAX_WIDTH:
        raise RuntimeError(f"{what}: {C} channels; at most {MAX_WIDTH}")
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"{what}: activation {activation!r}; supported: None, 'relu', 'silu'")
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if not t.is_cuda:
            raise RuntimeError(f"{what}: `{name}` lives on {t.device}; the kernels run only on a GPU (there is no CPU fallback)")
        if t.device != x.device:
            raise RuntimeError(f"{what}: `{name}` lives on {t.device}, x on {x.device}")
    if weight.shape != (C,) or bias.shape != (C,):
        raise RuntimeError(f"{what}: weight and bias must have shape ({C},)")


def _sizes(x):
    return (x.shape[0], 1, x.shape[1]) if x.dim() == 2 else tuple(x.shape)


def _out_dtype(x, out_dtype):
    if out_dtype is not None:
        return out_dtype
    return torch.float32 if torch.is_autocast_enabled() else x.dtype


def _per_utterance(what, x, lengths):
    if lengths is None:
        return None
    if x.dim() != 3:
        raise RuntimeError(f"{what}: lengths go with x of shape [batch, frames, channels]")
    return frames_of(what, "lengths", lengths, x, x.shape[0])


def _forward(x, num_groups, weight, bias, eps, activation, lengths, out_dtype, with_stats):
    """x, weight, bias dense; weight, bias float32."""
    N, T, C = _sizes(x)
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    stats = None
    if with_stats and (T > 1 or lengths is not None):
        stats = torch.empty((N, num_groups, 2), dtype=torch.float32, device=x.device)
    size = _lib.lib.lmufft_group_norm_workspace_bytes(N, T, C, num_groups, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    with on_device(x.device) as stream:
        rc = _lib.lib.lmufft_group_norm(x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), bias.data_ptr(), ptr(lengths), N, T,
                                        C, num_groups, eps, _ACTIVATIONS[activation], out.data_ptr(), _DTYPES[out_dtype],
                                        ptr(stats), ptr(ws), size, stream)
    if rc:
        _lib.check(rc, "lmufft_group_norm")
    return out, stats


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
               activation: Optional[str] = None, lengths: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(group_norm(x)) for x [B, T, C] (statistics over an utterance's frames) or [N, C] (of each row), no autograd.

    weight, bias: [C].  activation: None, "relu" or "silu".  lengths [B]: frames of each utterance (clamped to [0, T]).
    The result has `out_dtype`, by default float32 under autocast (where torch runs its norms in float32) and the input's
    dtype otherwise.  At most 1024 channels."""
    out_dtype = _out_dtype(x, out_dtype)
    _check("group_norm", x, num_groups, weight, bias, activation, out_dtype)
    lengths = _per_utterance("group_norm", x, lengths)
    return _forward(dense(x.detach()), num_groups, dense(weight.detach().float()), dense(bias.detach().float()), float(eps),
                    activation, lengths, out_dtype, False)[0]


class _GroupNormTrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lengths, num_groups, eps, activation, out_dtype):
        x, w, b = dense(x), dense(weight.float()), dense(bias.float())
        out, stats = _forward(x, num_groups, w, b, eps, activation, lengths, out_dtype, True)
        ctx.save_for_backward(x, w, b, lengths, stats)
        ctx.conf = (num_groups, eps, activation)
        ctx.params = (weight, bias)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, b, lengths, stats = ctx.saved_tensors
        num_groups, eps, activation = ctx.conf
        N, T, C = _sizes(x)
        if dy.dtype not in _DTYPES:
            dy = dy.float()
        dy = dense(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        # parameters of a GradBuckets: the kernel writes into the bucket and autograd adopts the slices as .grad
        slots = [grad_slot(p) for p in ctx.params]
        if any(s is None and hasattr(p, "_grad_view") for s, p in zip(slots, ctx.params)):
            run_deferred_sums()  # a gradient handed to autograd may be added into a slice that a deferred sum still owes
        dw, db = (torch.empty(C, dtype=torch.float32, device=x.device) if s is None else s for s in slots)
        size = _lib.lib.lmufft_group_norm_workspace_bytes(N, T, C, num_groups, 1)
        ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        with on_device(x.device) as stream:
            rc = _lib.lib.lmufft_group_norm_bwd(
                x.data_ptr(), _DTYPES[x.dtype], dy.data_ptr(), _DTYPES[dy.dtype], w.data_ptr(), b.data_ptr(), ptr(lengths),
                ptr(stats), N, T, C, num_groups, eps, _ACTIVATIONS[activation], dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                ptr(ws), size, stream)
        if rc:
            _lib.check(rc, "lmufft_group_norm_bwd")
        dw, db = (t.to(p.dtype) if s is None else adopt(t) for t, s, p in zip((dw, db), slots, ctx.params))
        return dx, dw, db, None, None, None, None, None


def group_norm_train(x: torch.Tensor, num_groups: int, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
                     activation: Optional[str] = None, lengths: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """group_norm with autograd for x, weight and bias (parameters of a GradBuckets get their gradients in place)."""
    out_dtype = _out_dtype(x, out_dtype)
    _check("group_norm_train", x, num_groups, weight, bias, activation, out_dtype)
    lengths = _per_utterance("group_norm_train", x, lengths)
    return _GroupNormTrain.apply(x, weight, bias, lengths, num_groups, float(eps), activation, out_dtype)
