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
zeros, and the state is the one behind the last frame inside.  An infinity or a NaN inside the length reaches the frames from
its own on (an infinity may come out as a NaN there), and none before.  The decays are constants of the model: no gradient is
returned for them, and the backward has no backward of its own.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._call import ops

SUPPORTED_HEAD_WIDTHS = (32, 64, 128)


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                    lengths: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Causal decay attention of q, k [B, T, heads * d_k] and v [B, T, heads * d_v] -> [B, T, heads * d_v].

    All float32 or all bfloat16; head widths 32, 64, 128.  log_decay: float32 [heads], the logarithm of each head's decay
    (0 keeps everything, -inf only the frame itself).  lengths [B]: frames of each utterance (whole numbers, clamped to
    [0, T]).  state: float32 [B, heads, d_k, d_v], contiguous; read as the state before the first frame and REPLACED by the
    state behind the last one, so the next call goes on from there.  scale: by default d_k ** -0.5.  Tensors may be column
    blocks of a wider one.  No autograd."""
    return ops.decay_attention(q, k, v, num_heads, log_decay, lengths, state, scale)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                         state: torch.Tensor, active: Optional[torch.Tensor] = None,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One frame of each stream: q, k [B, heads * d_k], v [B, heads * d_v] -> [B, heads * d_v]; `state` [B, heads, d_k,
    d_v] is updated in place.  Streams whose `active` [B] is 0 (or False) get zeros and keep their state.  The same operator
    as decay_attention with one frame; the calls may be mixed.  No autograd."""
    return ops.decay_attention_step(q, k, v, num_heads, log_decay, state, active, scale)


def decay_attention_train(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                          lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """decay_attention with autograd for q, k and v (states start at zero)."""
    return ops.decay_attention_train(q, k, v, num_heads, log_decay, lengths, scale)


def decay_attention_train_packed(qkv: torch.Tensor, num_heads: int, log_decay: torch.Tensor,
                                 lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """decay_attention_train with q, k, v given as the column blocks of one tensor [B, T, 3 * heads * width] (one projection
    over the concatenated weights); the gradient comes back as one tensor of that layout."""
    return ops.decay_attention_train_packed(qkv, num_heads, log_decay, lengths, scale)
