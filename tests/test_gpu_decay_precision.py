"""GPU tests of what the bf16 decay attention rounds before its result: nothing below sixteen bits, whatever the length of the
call, the batch around an utterance, or the place of a frame.

Tolerance.  A bf16 keeps 2^-8 of a value at worst, two of them 2^-16.  A term of an output passes through one score (two bf16
terms), or through the state: the scaled v that enters it and the state's copy that multiplies q, two terms each; so 2^-15 M
in all, M the sum of the terms' magnitudes; besides the 32-bit bound of tests/test_gpu_decay.py and half a step of the result,
2^-8 |ref|."""
import pytest
import torch

from oracle import decay_oracle as do
from tests.test_gpu_decay import _bound32, _decays, _dev, _make

pytestmark = pytest.mark.gpu


def _call(q, k, v, w, H, ld, lengths):
    """(out, dq, dk, dv) of the kernels."""
    from asr_amd.decay import decay_attention_train

    dev = _dev()
    ln = None if lengths is None else torch.tensor(lengths, device=dev)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = decay_attention_train(*leaves, H, ld.to(dev), ln)
    return out.detach(), *torch.autograd.grad(out, leaves, w.to(dev))


def _refs(q, k, v, w, ld, lengths):
    return do.decay_attention(q, k, v, ld, lengths)[0], *do.decay_attention_backward(q, k, v, w, ld, lengths)


def _tight(name, got, ref, M, T, d):
    err = (got.double().cpu() - ref).abs()
    over = err - (_bound32(M, T, d) + 2.0 ** -15 * M + 2.0 ** -8 * ref.abs())
    assert (over <= 0).all(), (name, float(over.max()), (over > 0).nonzero()[0].tolist())


@pytest.mark.parametrize("H,d,dv", [(5, 64, 64), (2, 32, 128), (3, 128, 128)])
def test_an_utterance_alone_and_in_a_padded_batch(H, d, dv):
    """The frames of a short utterance come out bit for bit the same whatever batch it lies in, and so do the first frames of a
    longer one (no state reaches them), within the tolerance."""
    T, lengths = 200, [200, 3, 70]
    q, k, v, w, _ = _make(3, T, H, d, dv, torch.bfloat16, 5)
    w, ld = w.to(torch.bfloat16), _decays(H)
    whole = _call(q, k, v, w, H, ld, lengths)
    for b, n in ((1, 3), (0, 32), (2, 20)):
        part = [t[b:b + 1, :n].contiguous() for t in (q, k, v, w)]
        alone = _call(*part, H, ld, None)
        assert torch.equal(whole[0][b:b + 1, :n], alone[0]) and torch.equal(whole[1][b:b + 1, :n], alone[1]), (b, n)
        if n == lengths[b]:
            assert all(torch.equal(x[b:b + 1, :n], y) for x, y in zip(whole, alone))
        size = [t.abs() for t in part]
        for name, got, r, m in zip(("out", "dq", "dk", "dv"), alone, _refs(*part, ld, None), _refs(*size, ld, None)):
            _tight(name, got, r, m, n, max(d, dv))


SHAPES = [
    # B, T, H, dk, dv, lengths
    (3, 200, 5, 64, 64, [200, 3, 70]),
    (2, 129, 2, 32, 128, None),
    (2, 150, 3, 128, 128, [150, 65]),
    (2, 333, 2, 128, 32, [333, 64]),
    (1, 1001, 5, 64, 64, None),         # several segments
    (1, 4000, 2, 32, 64, [3911]),       # joined by a launch of their own
]


@pytest.mark.parametrize("B,T,H,dk,dv,lengths", SHAPES)
def test_every_frame_without_a_state(B, T, H, dk, dv, lengths):
    q, k, v, w, _ = _make(B, T, H, dk, dv, torch.bfloat16, T)
    w, ld = w.to(torch.bfloat16), _decays(H)
    got = _call(q, k, v, w, H, ld, lengths)
    size = [t.abs() for t in (q, k, v, w)]
    for name, g, r, m in zip(("out", "dq", "dk", "dv"), got, _refs(q, k, v, w, ld, lengths), _refs(*size, ld, lengths)):
        _tight(name, g, r, m, T, max(dk, dv))


@pytest.mark.parametrize("B,T,H,dk,dv,lengths", SHAPES + [(4, 1, 6, 64, 64, None), (3, 50, 6, 64, 64, [50, 0, 7])])
def test_every_frame_from_a_state(B, T, H, dk, dv, lengths):
    from asr_amd.decay import decay_attention

    dev = _dev()
    q, k, v, _, st = _make(B, T, H, dk, dv, torch.bfloat16, T + 1)
    ld = _decays(H)
    ln = None if lengths is None else torch.tensor(lengths, device=dev)
    sd = st.to(dev)
    out = decay_attention(*(t.to(dev) for t in (q, k, v)), H, ld.to(dev), ln, sd)
    ref, S = do.decay_attention(q, k, v, ld, lengths, st)
    M, MS = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, lengths, st.abs())
    _tight("out", out, ref, M, T, dk)
    assert ((sd.double().cpu() - S).abs() <= _bound32(MS, T, 0)).all()
