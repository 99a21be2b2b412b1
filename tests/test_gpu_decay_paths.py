"""GPU tests of the causal decay attention's launch forms: ragged batches whose workgroups go from the longest utterance to the
shortest, long recordings whose segments' states are joined several a wave.  Each test first checks, by the workspace query and
the rule of the launch, that its sizes take the form it is about.  Oracle and tolerances are those of tests/test_gpu_decay.py."""
import math

import pytest
import torch

from oracle import decay_oracle as do
from tests.test_gpu_decay import _bound32, _close, _decays, _dev, _make

pytestmark = pytest.mark.gpu

CODE = {torch.float32: 0, torch.bfloat16: 1}


def _segments(dtype, B, T, H, dk, dv, backward):
    """Segments of an utterance: the workspace holds one state [dk][dv] for each of them, head and role, or nothing for one."""
    from asr_amd import _lib

    assert (_lib.F32, _lib.BF16) == (CODE[torch.float32], CODE[torch.bfloat16])
    n = _lib.lib.lmufft_decay_workspace_bytes(CODE[dtype], B, T, H, dk, dv, int(backward))
    one = 4 * (3 if backward else 1) * B * H * dk * dv
    assert n % one == 0
    return max(1, n // one)


def _ordered(dtype, B, T, H, dk, dv, backward):
    """More than 256 workgroups and 2 to 64 utterances with lengths."""
    return 1 < B <= 64 and B * H * (3 if backward else 1) * _segments(dtype, B, T, H, dk, dv, backward) > 256


def _ragged(B, T, kind):
    """Lengths in the order of the batch.  mixed: ties, nothing, everything, and values outside [0, T]."""
    if kind == "ties":
        return [T if b % 3 else T - 1 for b in range(B)]
    if kind == "one":
        return [0] * (B - 1) + [T]
    g = torch.Generator().manual_seed(B * 1000 + T)
    n = torch.randint(1, T + 1, (B,), generator=g).tolist()
    for i, x in enumerate((0, T, n[-1], T + 5, -3, 0, 1, T, n[-2], T // 2, T // 2)):
        if 3 * i < B:
            n[3 * i] = x
    return n


def _against_the_oracle(B, T, H, dk, dv, lengths, dtype, seed):
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    q, k, v, w, _ = _make(B, T, H, dk, dv, dtype, seed)
    ld = _decays(H, seed)
    ln = torch.tensor(lengths, dtype=torch.int32, device=dev)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = decay_attention_train(*leaves, H, ld.to(dev), ln)
    grads = torch.autograd.grad(out, leaves, w.to(dev))
    assert torch.equal(out.detach(), decay_attention(*leaves, H, ld.to(dev), ln))
    ref = (do.decay_attention(q, k, v, ld, lengths)[0], *do.decay_attention_backward(q, k, v, w, ld, lengths))
    size = [t.abs() for t in (q, k, v, w)]
    M = (do.decay_attention(*size[:3], ld, lengths)[0], *do.decay_attention_backward(*size, ld, lengths))
    for got, r, m, name in zip((out, *grads), ref, M, ("out", "dq", "dk", "dv")):
        _close(got, r, m, T, max(dk, dv), dtype, name)
        for b, n in enumerate(lengths):
            assert (got[b, min(max(n, 0), T):] == 0).all(), (name, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,dk,dv,kind,forward,backward", [
    (64, 130, 6, 32, 32, "mixed", True, True),
    (64, 70, 5, 32, 32, "ties", True, True),
    (64, 40, 5, 64, 32, "one", True, True),      # the backward's launches: two roles, then one
    (33, 130, 6, 64, 64, "mixed", False, True),
    (2, 70, 130, 32, 32, "mixed", True, True),
    (2, 70, 130, 32, 32, "one", True, True),
    (65, 70, 5, 32, 32, "mixed", False, False),  # more than a wave ranks: in the order of the batch
    (96, 130, 6, 32, 64, "mixed", False, False),
])
def test_ragged_batches(B, T, H, dk, dv, kind, forward, backward, dtype):
    assert _ordered(dtype, B, T, H, dk, dv, False) == forward
    # (unequal widths: a launch of two roles and one of the third; the third's alone is the smaller)
    roles = 3 if dk == dv else 1
    n = _segments(dtype, B, T, H, dk, dv, True)
    assert (1 < B <= 64 and B * H * roles * n > 256) == backward
    _against_the_oracle(B, T, H, dk, dv, _ragged(B, T, kind), dtype, T + B)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [2, 3, 31, 32, 63, 64])
def test_the_order_is_a_permutation(B, dtype):
    """Every utterance once, whatever the lengths' ties: each row against the same utterances in another order."""
    from asr_amd.decay import decay_attention

    dev = _dev()
    T, H = 50, max(5, -(-257 // B))
    assert _ordered(dtype, B, T, H, 32, 32, False)
    q, k, v, _, _ = (t.to(dev) for t in _make(B, T, H, 32, 32, dtype, B))
    ld = _decays(H, B).to(dev)
    for kind in ("mixed", "ties", "one"):
        ln = torch.tensor(_ragged(B, T, kind), device=dev)
        out = decay_attention(q, k, v, H, ld, ln)
        back = torch.arange(B - 1, -1, -1, device=dev)
        assert torch.equal(decay_attention(q[back], k[back], v[back], H, ld, ln[back])[back], out)
        plain = torch.cat([decay_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], H, ld, ln[b:b + 1]) for b in range(B)])
        assert torch.equal(plain, out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,dk,dv,lengths", [
    (4000, 2, 32, 32, None),
    (4000, 2, 32, 32, [1911]),        # ends inside a segment in the middle
    (4000, 2, 32, 32, [0]),
    (16500, 1, 32, 32, None),
    (16500, 1, 32, 64, [16385]),
])
def test_many_segments(T, H, dk, dv, lengths, dtype):
    from asr_amd.decay import decay_attention

    dev = _dev()
    n = _segments(dtype, 1, T, H, dk, dv, False)
    assert n >= 18  # a wave of the join holds several segments, and the last waves fewer
    q, k, v, w, st = _make(1, T, H, dk, dv, dtype, T)
    ld = torch.tensor([math.log1p(-2.0 ** -9), 0.0][:H])
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    a = [t.to(dev) for t in (q, k, v)]
    ref, _ = do.decay_attention(q, k, v, ld, lengths)
    M, _ = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, lengths)
    _close(decay_attention(*a, H, ld.to(dev), ln), ref, M, T, dk, dtype, "out")
    sd = st.to(dev)
    out = decay_attention(*a, H, ld.to(dev), ln, sd)
    ref, S = do.decay_attention(q, k, v, ld, lengths, st)
    M, MS = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, lengths, st.abs())
    _close(out, ref, M, T, dk, dtype, "out from a state")
    _close(sd, S, MS, T, 0, torch.float32, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[4000], [2049]])
def test_many_segments_backward(lengths, dtype):
    T, H, d = 4000, 2, 32
    assert _segments(dtype, 1, T, H, d, d, True) >= 18
    _against_the_oracle(1, T, H, d, d, lengths, dtype, 9)
