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
from ._call import ops

MAX_WIDTH = 1024


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
               activation: Optional[str] = None, lengths: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(group_norm(x)) for x [B, T, C] (statistics over an utterance's frames) or [N, C] (of each row), no autograd.

    x: float32 or bfloat16; weight, bias: [C].  activation: None, "relu" or "silu".  lengths [B]: frames of each utterance
    (whole numbers, clamped to [0, T]).  The result has `out_dtype`, by default float32 under autocast (where torch runs its
    norms in float32) and the input's dtype otherwise.  At most 1024 channels, and 65535 utterances (rows: any number)."""
    return ops.group_norm(x, num_groups, weight, bias, eps, activation, lengths, out_dtype)


def group_norm_train(x: torch.Tensor, num_groups: int, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-5,
                     activation: Optional[str] = None, lengths: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """group_norm with autograd for x, weight and bias (the backward has no backward of its own)."""
    return ops.group_norm_train(x, num_groups, weight, bias, eps, activation, lengths, out_dtype)
