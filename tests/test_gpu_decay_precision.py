"""GPU tests of what the bf16 decay attention rounds before its result: a score loses nothing above sixteen bits, whatever the
length of the call or the batch around an utterance.

Tolerance.  A bf16 keeps 2^-8 of a value at worst, two of them 2^-16, so a score in two terms loses 2^-16 M, M the sum of the
magnitudes of an output's terms; 2^-15 M is allowed, besides the 32-bit bound of tests/test_gpu_decay.py and half a step of the
result, 2^-8 |ref|."""
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
