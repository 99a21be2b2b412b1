"""GPU tests of the residual dropout (k_dropout_add): the decisions against the hash restated in the oracle, the values
against the arithmetic, and the block the new operators make together.

Tolerance of a value: x / (1 - p) and the sum are three roundings of 2^-24 each, the result's own type one of half a step."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a GPU")
    return torch.device("cuda:0")


def _keep(shape, p, seeds):
    C = shape[-1]
    rows = np.arange(int(np.prod(shape[:-1])), dtype=np.uint64)[:, None]
    return torch.from_numpy(ao.hash_keep(rows, np.arange(C, dtype=np.uint64)[None], C, p, *seeds).copy()).reshape(shape)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1,), (3, 1), (5, 2), (7, 3), (1, 8), (9, 17), (4, 33, 384), (2, 129, 385), (5, 1001), (300, 1000)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.75])
def test_values_and_gradients(shape, residual, dtype, p):
    from asr_amd.dropout import dropout_add

    dev = _dev()
    g = torch.Generator().manual_seed(len(shape) + shape[-1])
    x = torch.randn(*shape, generator=g).to(dtype)
    r = None if residual is None else torch.randn(*shape, generator=g).to(residual)
    seeds = (20240611, 0xFFFFFFF0)
    keep = _keep(shape, p, seeds)
    xd = x.to(dev).requires_grad_(True)
    rd = None if r is None else r.to(dev).requires_grad_(True)
    y = dropout_add(xd, rd, p, seeds)
    out = dtype if residual is None else torch.promote_types(dtype, residual)
    assert y.dtype == out
    ref = keep * x.double() / (1 - p) + (0 if r is None else r.double())
    size = keep * x.double().abs() / (1 - p) + (0 if r is None else r.double().abs())
    tol = 4 * 2.0 ** -24 * size + _half_step(out) * (ref.abs() + 4 * 2.0 ** -24 * size) + 1e-38
    assert ((y.detach().double().cpu() - ref).abs() <= tol).all()
    dy = torch.randn(*shape, generator=g).to(out)
    y.backward(dy.to(dev))
    ref = keep * dy.double() / (1 - p)
    assert ((xd.grad.double().cpu() - ref).abs() <= (4 * 2.0 ** -24 + _half_step(dtype) * 1.001) * ref.abs() + 1e-38).all()
    if rd is not None:
        assert torch.equal(rd.grad.cpu(), dy.to(residual))


def test_properties():
    from asr_amd import dropout

    dev = _dev()
    x = torch.ones(4096, 96, device=dev)
    y = dropout.dropout_add(x, None, 0.2, (1, 2))
    rate = (y != 0).float().mean().item()
    assert abs(rate - 0.8) < 4 * (0.16 / x.numel()) ** 0.5
    assert torch.equal(y, dropout.dropout_add(x, None, 0.2, (1, 2))) and not torch.equal(y, dropout.dropout_add(x, None, 0.2, (2, 2)))
    assert torch.equal(dropout.dropout_add(x.expand(2, 4096, 96), None, 0.2, (1, 2))[0], y)  # rows are counted on
    odd = torch.cat([x.new_zeros(4096, 1), x], -1)[:, 1:]
    assert torch.equal(dropout.dropout_add(odd, odd, 0.2, (1, 2)), y + 1)
    inf = torch.full((64, 96), float("inf"), device=dev)
    z = dropout.dropout_add(inf, None, 0.5, (3, 4))
    assert set(z.unique().tolist()) == {0.0, float("inf")}  # a dropped value is zero whatever it was
    torch.manual_seed(3)
    dropout._dropout_calls = 0
    a1, a2 = dropout.dropout_add(x), dropout.dropout_add(x)
    torch.manual_seed(3)
    dropout._dropout_calls = 0
    assert torch.equal(a1, dropout.dropout_add(x)) and not torch.equal(a1, a2)
    assert dropout.dropout_add(x[:0]).shape == (0, 96)
    for bad, kind, text in ((dict(p_drop=1.0), ValueError, "probability"), (dict(residual=x[:1]), RuntimeError, "does not match"),
                            (dict(residual=x.half()), RuntimeError, "supported dtypes"), (dict(residual=x.cpu()), RuntimeError, "no CPU"),
                            (dict(out_dtype=torch.float16), RuntimeError, "output dtype")):
        with pytest.raises(kind, match=text):
            dropout.dropout_add(x, **bad)
    with pytest.raises(RuntimeError, match="channels"):
        dropout.dropout_add(x[:, :0])


def test_replays_draw_fresh_masks_and_forward_agrees_with_backward():
    from asr_amd.dropout import bump_dropout_epoch, dropout_add, dropout_epoch

    dev = _dev()
    epoch = dropout_epoch(dev)
    x = torch.randn(64, 96, device=dev, requires_grad=True)
    dy = torch.ones(64, 96, device=dev)

    def step():
        bump_dropout_epoch(dev)
        y = dropout_add(x, None, 0.3, (5, 6))
        return y.detach(), *torch.autograd.grad(y, x, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y != 0, dx != 0)
        keep = _keep((64, 96), 0.3, (5, (6 + int(epoch.item())) & 0xFFFFFFFF))
        assert torch.equal(dx.cpu() != 0, keep)
        seen.append(keep)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_block_the_operators_make(dtype):
    """x + dropout(group_norm_silu(decay_attention(q, k, v))) and its gradients, against the three oracles in a row; then the
    same block frame by frame.  The tolerance is the sum of the steps': bf16 rounds each intermediate once (2^-8), the norm
    divides by a standard deviation and so passes on what comes in relative to its group."""
    from asr_amd.decay import decay_attention_step, decay_attention_train
    from asr_amd.dropout import dropout_add
    from asr_amd.groupnorm import group_norm, group_norm_train
    from oracle import decay_oracle, groupnorm_oracle

    dev = _dev()
    B, T, H, d = 2, 90, 6, 64
    C = H * d
    g = torch.Generator().manual_seed(17)
    x, q, k, v = (torch.randn(B, T, C, generator=g).to(dtype) for _ in range(4))
    w, b = 1 + 0.1 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g)
    ld = torch.log1p(-2.0 ** (-5 - torch.arange(H, dtype=torch.float32)))
    lengths, seeds, p = [90, 41], (7, 8), 0.1
    dy = torch.randn(B, T, C, generator=g).to(dtype)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, q, k, v, w, b)]
    xd, qd, kd, vd, wd, bd = leaves
    a = decay_attention_train(qd, kd, vd, H, ld.to(dev), torch.tensor(lengths, device=dev))
    n = group_norm_train(a.reshape(B * T, C), H, wd, bd, 1e-5, "silu").reshape(B, T, C)
    y = dropout_add(n, xd, p, seeds)
    grads = torch.autograd.grad(y, leaves, dy.to(dev))

    ra, _ = decay_oracle.decay_attention(q, k, v, ld, lengths)
    rn = groupnorm_oracle.group_norm(ra.reshape(B * T, C), H, w, b, 1e-5, "silu")
    keep = _keep((B, T, C), p, seeds)
    ry = x.double() + keep * rn.reshape(B, T, C) / (1 - p)
    dn = keep * dy.double() / (1 - p)
    da, dw, db = groupnorm_oracle.group_norm_backward(ra.reshape(B * T, C), H, w, b, dn.reshape(B * T, C), 1e-5, "silu")
    dqkv = decay_oracle.decay_attention_backward(q, k, v, da.reshape(B, T, C), ld, lengths)
    # 2-norm: the roundings of the chain add in quadrature, at most eight of half a step (32 bits: of the sums' 2^-24 sqrt(200))
    most = 8 ** 0.5 * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * 200 ** 0.5)
    for got, ref, name in zip((y, *grads), (ry, dy.double(), *dqkv, dw, db), ("y", "dx", "dq", "dk", "dv", "dw", "db")):
        rel = float((got.detach().double().cpu() - ref).norm() / ref.norm())
        assert rel <= most, (name, rel)
    # one frame at a time, as a stream is served
    st = torch.zeros(B, H, d, d, device=dev)
    with torch.no_grad():
        for t in range(lengths[1]):
            at = decay_attention_step(qd[:, t], kd[:, t], vd[:, t], H, ld.to(dev), st)
            yt = dropout_add(group_norm(at, H, wd, bd, 1e-5, "silu"), xd[:, t], 0.0)
            rel = float((yt.double().cpu() - (x[:, t].double() + rn.reshape(B, T, C)[:, t])).norm() / ry[:, t].norm())
            assert rel <= most, (t, rel)
