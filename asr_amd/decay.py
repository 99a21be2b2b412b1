"""Causal linear attention with one decay per head, on the GPU (HIP kernels k_decay, k_decay_states, k_decay_step).

Per head, with a decay lambda = exp(log_decay) in [0, 1] and a state S [d_k, d_v] (zeros at an utterance's start):

    S_t = lambda S_(t-1) + k_t v_t^T,      o_t = scale * S_t^T q_t

that is o_t = scale * sum_(j <= t) lambda^(t-j) (q_t . k_j) v_j: attention whose cost grows with the frames and not with
their square, and which runs as well frame by frame.  It takes the [batch, frames, heads * width] tensors that
masked_attention takes (asr_amd/attention.py), but is causal: frame t sees the frames up to t only.

    decay_attention               utterances, or the next frames of streams whose states go on (no autograd)
    decay_attention_step          one frame of each stream, the states updated in place (no autograd)
    decay_attention_train         with autograd for q, k, v
    decay_attention_train_packed  the same on q | k | v as the column blocks of one projection's output

Frames from an utterance's length on are padding: whatever they hold, they are not read, their outputs and gradients are
zeros, and the state is the one behind the last frame inside.  (A frame INSIDE the length that holds inf or NaN spreads it
to all later frames, and may spread it to the up to 63 frames before it that share its chunk.)  The decays are constants of
the model: no gradient is returned for them.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._call import dense, frames_of, on_device, ptr

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
SUPPORTED_HEAD_WIDTHS = (32, 64, 128)


def _check(what: str, q, k, v, num_heads: int, log_decay, dims: int):
    """(d_k, d_v) of the call, or the error that says what is wrong with it."""
    dt = q.dtype
    if dt not in _DTYPES or k.dtype != dt or v.dtype != dt:
        raise RuntimeError(f"{what}: dtypes {q.dtype}, {k.dtype}, {v.dtype}; supported: all float32 or all bfloat16")
    if q.dim() != dims or k.shape != q.shape or v.dim() != dims or v.shape[:-1] != q.shape[:-1]:
        raise RuntimeError(f"{what}: q and k must share one {'[batch, frames, channels]' if dims == 3 else '[batch, channels]'} "
                           f"shape and v its leading dimensions, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    dev = q.device
    for name, t in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay)):
        if not t.is_cuda:
            raise RuntimeError(f"{what}: `{name}` lives on {t.device}; the kernels run only on a GPU (there is no CPU fallback)")
        if t.device != dev:
            raise RuntimeError(f"{what}: `{name}` lives on {t.device}, q on {dev}")
    c, cv = q.shape[-1], v.shape[-1]
    if num_heads <= 0 or c % num_heads or cv % num_heads:
        raise RuntimeError(f"{what}: {c} and {cv} channels do not split into {num_heads} heads")
    dk, dv = c // num_heads, cv // num_heads
    if dk not in SUPPORTED_HEAD_WIDTHS or dv not in SUPPORTED_HEAD_WIDTHS:
        raise RuntimeError(f"{what}: head widths {dk}, {dv}; supported: {SUPPORTED_HEAD_WIDTHS}")
    if log_decay.dtype != torch.float32 or log_decay.shape != (num_heads,):
        raise RuntimeError(f"{what}: log_decay must be float32 [{num_heads}], got {log_decay.dtype} {tuple(log_decay.shape)}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: the decays are constants; log_decay must not require a gradient")
    return dk, dv


def _check_state(what: str, state, q, B: int, H: int, dk: int, dv: int) -> None:
    if (state.dtype != torch.float32 or state.shape != (B, H, dk, dv) or not state.is_contiguous() or state.device != q.device
            or state.data_ptr() % 16):
        raise RuntimeError(f"{what}: `state` must be a contiguous float32 tensor [{B}, {H}, {dk}, {dv}] on {q.device} that starts "
                           f"on a 16-byte boundary, got {state.dtype} {tuple(state.shape)} on {state.device}")
    if state.requires_grad:
        raise RuntimeError(f"{what}: `state` is replaced in place and must not require a gradient")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [B, T, C] with rows the kernels can load 16 bytes at a time; a column block of a wider tensor stays in place."""
    per = 16 // t.element_size()
    if t.stride(2) == 1 and t.stride(1) % per == 0 and t.stride(0) % per == 0 and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(what, q, k, v, num_heads, dk, dv, log_decay, lengths, state, scale):
    B, T, _ = q.shape
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    dt = _DTYPES[q.dtype]
    out = torch.empty((B, T, num_heads * dv), dtype=q.dtype, device=q.device)
    size = _lib.lib.lmufft_decay_workspace_bytes(dt, B, T, num_heads, dk, dv, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    with on_device(q.device) as stream:
        rc = _lib.lib.lmufft_decay_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, q.stride(1), q.stride(0), k.stride(1), k.stride(0), v.stride(1),
            v.stride(0), log_decay.data_ptr(), ptr(lengths), B, T, num_heads, dk, dv, scale, out.data_ptr(), num_heads * dv,
            T * num_heads * dv, ptr(state), ptr(ws), size, stream)
    if rc:
        _lib.check(rc, "lmufft_decay_attention")
    return out


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                    lengths: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Causal decay attention of q, k [B, T, heads * d_k] and v [B, T, heads * d_v] -> [B, T, heads * d_v].

    log_decay: float32 [heads], the logarithm of each head's decay (0 keeps everything, -inf only the frame itself).
    lengths: frames of each utterance (clamped to [0, T]).  state: float32 [B, heads, d_k, d_v], contiguous; read as the
    state before the first frame and REPLACED by the state behind the last one, so the next call goes on from there.
    scale: by default d_k ** -0.5.  Tensors may be column blocks of a wider one.  No autograd."""
    dk, dv = _check("decay_attention", q, k, v, num_heads, log_decay, 3)
    B = q.shape[0]
    if state is not None:
        _check_state("decay_attention", state, q, B, num_heads, dk, dv)
    lengths = frames_of("decay_attention", "lengths", lengths, q, B)
    return _forward("decay_attention", q.detach(), k.detach(), v.detach(), num_heads, dk, dv, log_decay.detach(), lengths, state,
                    dk ** -0.5 if scale is None else float(scale))


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                         state: torch.Tensor, active: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One frame of each stream: q, k [B, heads * d_k], v [B, heads * d_v] -> [B, heads * d_v]; `state` [B, heads, d_k,
    d_v] is updated in place.  Streams whose `active` [B] is 0 (or False) get zeros and keep their state.  The same numbers
    as decay_attention with one frame; the calls may be mixed.  No autograd."""
    dk, dv = _check("decay_attention_step", q, k, v, num_heads, log_decay, 2)
    B = q.shape[0]
    _check_state("decay_attention_step", state, q, B, num_heads, dk, dv)
    active = frames_of("decay_attention_step", "active", active, q, B)
    q, k, v = (t if t.stride(1) == 1 else t.contiguous() for t in (q, k, v))
    log_decay = log_decay.contiguous()
    out = torch.empty((B, num_heads * dv), dtype=q.dtype, device=q.device)
    with on_device(q.device) as stream:
        rc = _lib.lib.lmufft_decay_attention_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPES[q.dtype], q.stride(0), k.stride(0), v.stride(0),
            log_decay.data_ptr(), ptr(active), B, num_heads, dk, dv, dk ** -0.5 if scale is None else float(scale),
            out.data_ptr(), num_heads * dv, state.data_ptr(), stream)
    if rc:
        _lib.check(rc, "lmufft_decay_attention_step")
    return out


def _backward(q, k, v, dout, num_heads, dk, dv, log_decay, lengths, scale, dq, dkey, dval):
    B, T, _ = q.shape
    dt = _DTYPES[q.dtype]
    if dout.dtype != q.dtype:
        dout = dout.to(q.dtype)
    dout = _rows(dout)
    size = _lib.lib.lmufft_decay_workspace_bytes(dt, B, T, num_heads, dk, dv, 1)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    with on_device(q.device) as stream:
        rc = _lib.lib.lmufft_decay_attention_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), dt, q.stride(1), q.stride(0), k.stride(1), k.stride(0),
            v.stride(1), v.stride(0), dout.stride(1), dout.stride(0), log_decay.data_ptr(), ptr(lengths), B, T, num_heads, dk,
            dv, scale, dq.data_ptr(), dkey.data_ptr(), dval.data_ptr(), dq.stride(1), dq.stride(0), dkey.stride(1),
            dkey.stride(0), dval.stride(1), dval.stride(0), ptr(ws), size, stream)
    if rc:
        _lib.check(rc, "lmufft_decay_attention_bwd")


class _DecayTrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, lengths, num_heads, dk, dv, scale):
        q, k, v = _rows(q), _rows(k), _rows(v)
        ctx.save_for_backward(q, k, v, log_decay, lengths)
        ctx.conf = (num_heads, dk, dv, scale)
        return _forward("decay_attention_train", q, k, v, num_heads, dk, dv, log_decay, lengths, None, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, log_decay, lengths = ctx.saved_tensors
        num_heads, dk, dv, scale = ctx.conf
        dq, dkey, dval = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        _backward(q, k, v, dout, num_heads, dk, dv, log_decay, lengths, scale, dq, dkey, dval)
        return dq, dkey, dval, None, None, None, None, None, None


class _DecayTrainPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, log_decay, lengths, num_heads, dk, scale):
        qkv = _rows(qkv)
        ctx.save_for_backward(qkv, log_decay, lengths)
        ctx.conf = (num_heads, dk, scale)
        q, k, v = qkv.chunk(3, dim=-1)
        return _forward("decay_attention_train_packed", q, k, v, num_heads, dk, dk, log_decay, lengths, None, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, log_decay, lengths = ctx.saved_tensors
        num_heads, dk, scale = ctx.conf
        grad = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _backward(*qkv.chunk(3, dim=-1), dout, num_heads, dk, dk, log_decay, lengths, scale, *grad.chunk(3, dim=-1))
        return grad, None, None, None, None, None


def decay_attention_train(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                          lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """decay_attention with autograd for q, k and v (states start at zero)."""
    dk, dv = _check("decay_attention_train", q, k, v, num_heads, log_decay, 3)
    lengths = frames_of("decay_attention_train", "lengths", lengths, q, q.shape[0])
    return _DecayTrain.apply(q, k, v, log_decay.contiguous(), lengths, num_heads, dk, dv,
                             dk ** -0.5 if scale is None else float(scale))


def decay_attention_train_packed(qkv: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                                 lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """decay_attention_train with q, k, v given as the column blocks of one tensor [B, T, 3 * heads * width] (one projection
    over the concatenated weights); the gradient comes back as one tensor of that layout."""
    if qkv.dim() != 3 or qkv.shape[2] % 3:
        raise RuntimeError(f"decay_attention_train_packed: qkv must be [batch, frames, 3 * channels], got {tuple(qkv.shape)}")
    q, k, v = qkv.detach().chunk(3, dim=-1)
    dk, _ = _check("decay_attention_train_packed", q, k, v, num_heads, log_decay, 3)
    lengths = frames_of("decay_attention_train_packed", "lengths", lengths, qkv, qkv.shape[0])
    return _DecayTrainPacked.apply(qkv, log_decay.contiguous(), lengths, num_heads, dk,
                                   dk ** -0.5 if scale is None else float(scale))
