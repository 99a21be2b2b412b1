"""Causal linear attention with a decay per head, frame by frame in 64 bits.  TEST INFRASTRUCTURE ONLY.

    S_t = lambda S_(t-1) + k_t v_t^T,   o_t = scale S_t^T q_t     (lambda = exp(log_decay) per head)

The gradients come from the adjoint recurrence G_t = lambda G_(t+1) + scale q_t do_t^T; tests/test_decay_oracle.py holds
them against autograd of the defining double sum and against differences.
"""
import torch


def _split(t, heads):
    t = t.double()
    return t.reshape(*t.shape[:2], heads, -1)


def decay_attention(q, k, v, log_decay, lengths=None, state=None, scale=None):
    """(out [B, T, H dv], state [B, H, dk, dv]) in float64."""
    H = log_decay.numel()
    q, k, v = _split(q, H), _split(k, H), _split(v, H)
    B, T, _, dk = q.shape
    dv = v.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    lam = torch.exp(log_decay.double())[None, :, None, None]
    lengths = [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if state is None else state.double().clone()
    out = torch.zeros(B, T, H, dv, dtype=torch.float64)
    n = torch.tensor(lengths)
    for t in range(T):
        b = (n > t).nonzero()[:, 0]
        S[b] = lam * S[b] + k[b, t, :, :, None] * v[b, t, :, None, :]
        out[b, t] = scale * (q[b, t, :, :, None] * S[b]).sum(2)
    return out.reshape(B, T, H * dv), S


def decay_attention_backward(q, k, v, dout, log_decay, lengths=None, scale=None):
    """(dq, dk, dv) in float64 for states that start at zero."""
    H = log_decay.numel()
    q, k, v, do = _split(q, H), _split(k, H), _split(v, H), _split(dout, H)
    B, T, _, dk = q.shape
    dv = v.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    lam = torch.exp(log_decay.double())[None, :, None, None]
    n = torch.tensor([T] * B if lengths is None else [min(max(int(x), 0), T) for x in lengths])
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64)
    dq, dkey, dval = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T):
        b = (n > t).nonzero()[:, 0]
        S[b] = lam * S[b] + k[b, t, :, :, None] * v[b, t, :, None, :]
        dq[b, t] = scale * (S[b] * do[b, t, :, None, :]).sum(3)
    G = torch.zeros_like(S)
    for t in range(T - 1, -1, -1):
        b = (n > t).nonzero()[:, 0]
        G[b] = lam * G[b] + scale * q[b, t, :, :, None] * do[b, t, :, None, :]
        dkey[b, t] = (G[b] * v[b, t, :, None, :]).sum(3)
        dval[b, t] = (G[b] * k[b, t, :, :, None]).sum(2)
    return dq.reshape(B, T, H * dk), dkey.reshape(B, T, H * dk), dval.reshape(B, T, H * dv)
