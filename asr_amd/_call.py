"""What the bindings of single operators share: the device and stream of a call, and the layouts its kernels read."""
from __future__ import annotations

import torch


class on_device:
    """The device of a call made current for it, and its stream there: `with on_device(x.device) as stream`.  (A guard that
    switches to the device that is current already would cost microseconds a call.)"""

    def __init__(self, device):
        self.device = device
        self.guard = None

    def __enter__(self):
        if torch.cuda.current_device() != self.device.index:
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def ptr(t):
    return None if t is None else t.data_ptr()


def dense(t: torch.Tensor) -> torch.Tensor:
    """`t` contiguous from a 16-byte boundary on."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def frames_of(what: str, name: str, counts, like: torch.Tensor, batch: int):
    """`counts` [batch] (frames of each utterance, or which streams are live) as the kernels read it: int32 on the device
    of `like`."""
    if counts is None:
        return None
    if counts.shape != (batch,):
        raise RuntimeError(f"{what}: `{name}` must have shape ({batch},), got {tuple(counts.shape)}")
    if counts.is_floating_point() or counts.is_complex():
        raise RuntimeError(f"{what}: `{name}` must hold whole numbers, got {counts.dtype}")
    if counts.dtype != torch.int32 or counts.device != like.device or not counts.is_contiguous():
        counts = counts.to(device=like.device, dtype=torch.int32).contiguous()
    return counts
