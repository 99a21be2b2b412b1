"""GPU test of the residual dropout on more elements than one launch has threads for (16384 workgroups of 256 threads, eight
elements each): every element against the hash restated in the oracle and the arithmetic in 64 bits."""
import pytest
import torch

from tests.test_gpu_dropout_add import _dev, _half_step, _keep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,C", [(35000, 1000), (34999, 1001)])
def test_more_elements_than_threads(rows, C):
    from asr_amd.dropout import dropout_add

    dev = _dev()
    assert rows * C > 16384 * 256 * 8
    g = torch.Generator(device=dev).manual_seed(C)
    x = torch.randn(rows, C, generator=g, device=dev).bfloat16().requires_grad_(True)
    r = torch.randn(rows, C, generator=g, device=dev)
    p, seeds = 0.25, (11, 12)
    y = dropout_add(x, r, p, seeds)
    dy = torch.randn(rows, C, generator=g, device=dev)
    dx, = torch.autograd.grad(y, x, dy)
    # (three roundings of 2^-24 and the gradient's half step, as in tests/test_gpu_dropout_add.py)
    for at in range(0, rows, 5000):
        part = slice(at, min(at + 5000, rows))
        keep = _keep_rows(part.start, part.stop, C, p, seeds).to(dev)
        kept = keep * x.detach()[part].double() / (1 - p)
        ref = kept + r[part].double()
        assert ((y.detach()[part].double() - ref).abs() <= 8 * 2.0 ** -24 * (kept.abs() + r[part].double().abs()) + 1e-38).all(), at
        ref = keep * dy[part].double() / (1 - p)
        assert ((dx[part].double() - ref).abs() <= (4 * 2.0 ** -24 + _half_step(torch.bfloat16) * 1.001) * ref.abs() + 1e-38).all(), at
    assert torch.equal(_keep((3, C), p, seeds), _keep_rows(0, 3, C, p, seeds))


def _keep_rows(first, last, C, p, seeds):
    """The decisions of rows first..last-1."""
    import numpy as np

    from oracle import attention_oracle as ao

    rows = np.arange(first, last, dtype=np.uint64)[:, None]
    return torch.from_numpy(ao.hash_keep(rows, np.arange(C, dtype=np.uint64)[None], C, p, *seeds).copy())
