"""CPU: the 64-bit oracle of the group norm against torch's group norm and autograd; refusals of the group norm and the
residual dropout that need no GPU."""
import ctypes

import pytest
import torch

from oracle import groupnorm_oracle as go


@pytest.mark.parametrize("activation", [None, "relu", "silu"])
def test_oracle_is_torch_group_norm(activation):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 7, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(3, 7, 12, generator=g, dtype=torch.float64)
    act = {None: lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu}[activation]
    lengths = [7, 3, 0]
    whole = act(torch.nn.functional.group_norm(x.transpose(1, 2), 4, w, b)).transpose(1, 2)
    assert torch.allclose(go.group_norm(x.detach(), 4, w.detach(), b.detach(), activation=activation), whole.detach(), rtol=1e-10)
    parts = [act(torch.nn.functional.group_norm(x[i:i + 1, :n].transpose(1, 2), 4, w, b)).transpose(1, 2) for i, n in enumerate(lengths) if n]
    y = go.group_norm(x.detach(), 4, w.detach(), b.detach(), activation=activation, lengths=lengths)
    assert torch.allclose(y[1, :3], parts[1][0].detach(), rtol=1e-10) and (y[1, 3:] == 0).all() and (y[2] == 0).all()
    loss = sum((p * dy[i:i + 1, :p.shape[1]]).sum() for i, p in enumerate(parts))
    ref = torch.autograd.grad(loss, (x, w, b))
    mine = go.group_norm_backward(x.detach(), 4, w.detach(), b.detach(), dy, activation=activation, lengths=lengths)
    for a, r in zip(mine, ref):
        assert torch.allclose(a, r, rtol=1e-9, atol=1e-12)
    # rows: every one a sample of its own
    rows = x.detach().reshape(21, 12)
    ref = act(torch.nn.functional.group_norm(rows, 4, w, b)).detach()
    assert torch.allclose(go.group_norm(rows, 4, w.detach(), b.detach(), activation=activation), ref, rtol=1e-10)


def test_python_refusals_on_the_cpu():
    from asr_amd.dropout import dropout_add
    from asr_amd.groupnorm import group_norm, group_norm_train

    x, w = torch.zeros(2, 5, 96), torch.zeros(96)
    for f in (group_norm, group_norm_train):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(x, 4, w, w)
        with pytest.raises(RuntimeError, match="do not split"):
            f(x, 5, w, w)
        with pytest.raises(RuntimeError, match="do not split"):
            f(x, 0, w, w)
        with pytest.raises(RuntimeError, match="activation"):
            f(x, 4, w, w, activation="tanh")
        with pytest.raises(RuntimeError, match="dtypes"):
            f(x.half(), 4, w, w)
        with pytest.raises(RuntimeError, match="must be"):
            f(x[0, 0], 4, w, w)
        with pytest.raises(RuntimeError, match="at most"):
            f(torch.zeros(2, 1028), 4, w, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dropout_add(x, x)
    with pytest.raises(RuntimeError, match="supported dtypes"):
        dropout_add(x.half())


def test_c_entry_points_refuse_before_any_launch():
    from asr_amd import _lib

    lib = _lib.lib
    p = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused
    q = ctypes.c_void_p(4100)

    def fwd(x=p, dt=_lib.F32, N=2, T=5, C=96, G=4, act=0, out=p, od=_lib.F32, ws=None, n=0):
        return lib.lmufft_group_norm(x, dt, p, p, None, N, T, C, G, 1e-5, act, out, od, None, ws, n, None)

    for call, text in ((dict(dt=3), b"dtype"), (dict(od=-1), b"dtype"), (dict(C=97), b"bad shape"), (dict(G=0), b"bad shape"),
                       (dict(N=-1), b"bad shape"), (dict(C=1028), b"at most"), (dict(act=3), b"activation"), (dict(x=None), b"NULL"),
                       (dict(out=None), b"NULL"), (dict(x=q), b"16-byte"), (dict(T=5000), b"workspace"), (dict(T=5000, ws=p, n=8), b"workspace"),
                       (dict(N=70000), b"utterances"), (dict(N=1, T=(1 << 30) + 1, C=1, G=1), b"frames")):
        assert fwd(**call) != 0 and text in lib.lmufft_last_error(), (call, lib.lmufft_last_error())
    assert fwd(N=0) == 0 and fwd(T=0) == 0
    assert lib.lmufft_group_norm_workspace_bytes(2, 5, 96, 5, 0) == 0
    assert lib.lmufft_group_norm_workspace_bytes(70000, 1, 96, 4, 0) == 0 and lib.lmufft_group_norm_workspace_bytes(70000, 1, 96, 4, 1) > 0
    rc = lib.lmufft_group_norm_bwd(p, 0, p, 0, p, p, None, None, 2, 5, 96, 4, 1e-5, 0, p, p, p, None, 0, None)
    assert rc != 0 and b"NULL" in lib.lmufft_last_error()  # no statistics
    rc = lib.lmufft_group_norm_bwd(p, 0, p, 0, p, p, None, p, 2, 5, 96, 4, 1e-5, 0, p, p, None, None, 0, None)
    assert rc != 0 and b"NULL" in lib.lmufft_last_error()

    def drop(x=p, xd=0, r=None, rd=0, rows=4, C=6, pd=0.1, out=p, od=0):
        return lib.lmufft_dropout_add(x, xd, r, rd, rows, C, pd, 1, 2, out, od, None)

    for call, text in ((dict(pd=1.0), b"probability"), (dict(pd=float("nan")), b"probability"), (dict(xd=5), b"dtype"), (dict(rows=-1), b"bad shape"),
                       (dict(C=0), b"bad shape"), (dict(rows=1 << 61), b"bad shape"), (dict(x=None), b"NULL"), (dict(out=q), b"16-byte"),
                       (dict(out=p, od=1), b"alias"), (dict(r=q), b"16-byte")):
        assert drop(**call) != 0 and text in lib.lmufft_last_error(), (call, lib.lmufft_last_error())
    assert drop(rows=0) == 0
