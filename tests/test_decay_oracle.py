"""CPU: the 64-bit oracle of the causal decay attention against the defining double sum, autograd and differences;
and the refusals of the entry points that need no GPU."""
import ctypes

import pytest
import torch

from oracle import decay_oracle as do


def _double_sum(q, k, v, log_decay, scale):
    B, T, C = q.shape
    H = log_decay.numel()
    split = lambda t: t.view(B, T, H, -1).transpose(1, 2)  # noqa: E731
    gap = torch.arange(T)[:, None] - torch.arange(T)[None, :]
    D = torch.where(gap >= 0, torch.exp(log_decay)[:, None, None] ** gap.clamp(min=0), 0.0)
    P = split(q) @ split(k).transpose(-1, -2) * D
    return (scale * P @ split(v)).transpose(1, 2).reshape(B, T, -1)


def _inputs(B=2, T=9, H=2, dk=4, dv=3):
    g = torch.Generator().manual_seed(1)
    mk = lambda d: torch.randn(B, T, H * d, generator=g, dtype=torch.float64)  # noqa: E731
    return mk(dk), mk(dk), mk(dv), torch.tensor([-0.3, 0.0], dtype=torch.float64)


def test_oracle_is_the_double_sum_and_its_autograd():
    q, k, v, ld = _inputs()
    for t in (q, k, v):
        t.requires_grad_(True)
    ref = _double_sum(q, k, v, ld, 0.5)
    out, _ = do.decay_attention(q.detach(), k.detach(), v.detach(), ld, scale=0.5)
    assert torch.allclose(out, ref.detach(), rtol=1e-12, atol=1e-12)
    w = torch.randn(ref.shape, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    grads = torch.autograd.grad(ref, (q, k, v), w)
    mine = do.decay_attention_backward(q.detach(), k.detach(), v.detach(), w, ld, scale=0.5)
    for a, b in zip(mine, grads):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_oracle_gradients_against_differences_with_lengths():
    q, k, v, ld = _inputs()
    lengths = [9, 4]
    w = torch.randn(2, 9, 6, dtype=torch.float64, generator=torch.Generator().manual_seed(3))
    mine = do.decay_attention_backward(q, k, v, w, ld, lengths)
    f = lambda *a: float((do.decay_attention(*a, ld, lengths)[0] * w).sum())  # noqa: E731
    h = 1e-5
    for which, at in ((0, (0, 3, 1)), (1, (1, 2, 5)), (2, (0, 8, 2)), (1, (1, 6, 0)), (2, (1, 3, 5))):
        up, dn = [q.clone(), k.clone(), v.clone()], [q.clone(), k.clone(), v.clone()]
        up[which][at] += h
        dn[which][at] -= h
        assert abs((f(*up) - f(*dn)) / (2 * h) - float(mine[which][at])) < 1e-7


def test_oracle_goes_on_from_a_state():
    q, k, v, ld = _inputs(T=11)
    whole, S = do.decay_attention(q, k, v, ld)
    a, mid = do.decay_attention(q[:, :4], k[:, :4], v[:, :4], ld)
    b, end = do.decay_attention(q[:, 4:], k[:, 4:], v[:, 4:], ld, state=mid)
    assert torch.allclose(torch.cat([a, b], 1), whole, rtol=1e-12, atol=1e-12) and torch.allclose(end, S, rtol=1e-12)


def test_python_refusals_on_the_cpu():
    from asr_amd import decay

    x, ld = torch.zeros(2, 5, 128), torch.zeros(2)
    st = torch.zeros(2, 2, 64, 64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        decay.decay_attention(x, x, x, 2, ld)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        decay.decay_attention_train(x, x, x, 2, ld)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        decay.decay_attention_step(x[:, 0], x[:, 0], x[:, 0], 2, ld, st)
    with pytest.raises(RuntimeError, match="dtypes"):
        decay.decay_attention(x.half(), x.half(), x.half(), 2, ld)
    with pytest.raises(RuntimeError, match="dtypes"):
        decay.decay_attention(x, x.bfloat16(), x, 2, ld)
    with pytest.raises(RuntimeError, match="share one"):
        decay.decay_attention(x, x[:, :4], x, 2, ld)
    with pytest.raises(RuntimeError, match="3 \\* channels"):
        decay.decay_attention_train_packed(x[..., :127], 1, ld)


def test_c_entry_points_refuse_before_any_launch():
    from asr_amd import _lib

    lib = _lib.lib
    p = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused
    fwd = lambda q=p, dt=_lib.BF16, ld=128, bs=640, B=2, T=5, H=2, dk=64, dv=64, ldo=128, st=None, ws=None, n=0, dec=p: (  # noqa: E731
        lib.lmufft_decay_attention(q, p, p, dt, ld, bs, 128, 640, 128, 640, dec, None, B, T, H, dk, dv, 0.125, p, ldo, 640, st,
                                   ws, n, None))
    for call, text in ((dict(dt=7), b"dtype"), (dict(dk=48), b"head widths"), (dict(dv=256), b"head widths"),
                       (dict(B=-1), b"bad shape"), (dict(H=0), b"bad shape"), (dict(q=None), b"`q` is NULL"),
                       (dict(ld=130), b"16-byte"), (dict(q=ctypes.c_void_p(4104)), b"16-byte"), (dict(ld=-128), b"negative"),
                       (dict(ldo=64), b"overlap"), (dict(dec=None), b"log_decay"), (dict(st=ctypes.c_void_p(4100)), b"`state`"),
                       (dict(T=4000, B=1), b"workspace"), (dict(T=1 << 27), b"too large"), (dict(T=(1 << 25) + 1, B=1), b"too large"),
                       (dict(B=1 << 22, H=2, T=1), b"too large")):
        assert fwd(**call) != 0 and text in lib.lmufft_last_error(), (call, lib.lmufft_last_error())
    assert fwd(B=0) == 0 and fwd(T=0) == 0
    assert lib.lmufft_decay_workspace_bytes(_lib.BF16, 1, 4000, 2, 64, 64, 0) > 0
    assert lib.lmufft_decay_workspace_bytes(_lib.BF16, 1, 4000, 2, 60, 64, 0) == 0
    assert lib.lmufft_decay_workspace_bytes(_lib.BF16, 512, 4000, 2, 64, 64, 1) == 0
    rc = lib.lmufft_decay_attention_step(p, p, p, _lib.F32, 128, 128, 128, p, None, 2, 2, 64, 64, 0.125, p, 64, p, None)
    assert rc != 0 and b"row stride" in lib.lmufft_last_error()
    rc = lib.lmufft_decay_attention_step(p, p, p, _lib.F32, 128, 128, 128, p, None, 2, 2, 64, 64, 0.125, p, 128, None, None)
    assert rc != 0 and b"NULL" in lib.lmufft_last_error()
    rc = lib.lmufft_decay_attention_bwd(p, p, p, p, _lib.F32, *[640, 3200] * 4, p, None, 2, 5, 2, 64, 64, 0.125, p, p, p, 64, 640,
                                        128, 640, 128, 640, None, 0, None)
    assert rc != 0 and b"`dq` overlap" in lib.lmufft_last_error()
