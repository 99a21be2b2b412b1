"""GPU tests of the group norm with a result of another type than its input (as under autocast) and with more rows than the
kernels launch workgroups for, against the 64-bit oracle; tolerances as in tests/test_gpu_groupnorm.py."""
import pytest
import torch

from oracle import groupnorm_oracle as go
from tests.test_gpu_groupnorm import U, _dev, _make, _pieces, _within

pytestmark = pytest.mark.gpu


def _check(shape, groups, lengths, activation, dtype, out_dtype, autocast=False):
    from asr_amd.groupnorm import group_norm_train

    dev = _dev()
    x, w, b, dy = _make(shape, dtype, shape[0] * 5 + groups)
    hat, rstd, z, A, mean = _pieces(x.double(), groups, w.double(), b.double(), lengths)
    if activation == "relu":
        dy = torch.where(z.abs() < 1e-4, 0.0, dy.double()).float()
    dy = dy.to(out_dtype)
    ln = None if lengths is None else torch.tensor(lengths, device=dev)
    leaves = [x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)]
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        y = group_norm_train(leaves[0], groups, *leaves[1:], 1e-5, activation, ln, None if autocast else out_dtype)
    assert y.dtype == out_dtype
    grads = torch.autograd.grad(y, leaves, dy.to(dev))
    assert grads[0].dtype == dtype

    E = 160 + (shape[1] if len(shape) == 3 else 1) + shape[0]
    w, b, dyd = w.double(), b.double(), dy.double()
    h = E * U * (hat.abs() + A * rstd)
    soft = (2 * z.abs() + 20) * U
    ref = go.group_norm(x, groups, w, b, 1e-5, activation, lengths)
    _within(y, ref, 1.1 * w.abs() * h + soft * (z.abs() + b.abs()), out_dtype, "y")
    rx, rw, rb = go.group_norm_backward(x, groups, w, b, dyd, 1e-5, activation, lengths)
    s = torch.sigmoid(z)
    dz = dyd * {None: torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[activation]
    g, dyw = dz * w, (dyd * w).abs()
    tol = rstd * (E * U * (g.abs() + mean(g.abs()) + hat.abs() * mean((g * hat).abs())) + h * (mean(g * hat).abs() + dyw)
                  + mean(dyw * h) * (1 + hat.abs()) + soft * dyw)
    _within(grads[0], rx, tol, dtype, "dx")
    inside = (rstd > 0).double()
    flat = lambda t: (t * inside).reshape(-1, shape[-1]).sum(0)  # noqa: E731
    slope_err = 0.5 * w.abs() * h + soft
    _within(grads[1], rw, flat(E * U * (dz * hat).abs() + dz.abs() * h + (dyd * hat).abs() * slope_err), torch.float32, "dweight")
    _within(grads[2], rb, flat(E * U * dz.abs() + dyd.abs() * slope_err), torch.float32, "dbias")


SHAPES = [
    ((501, 384), 32, None),               # rows
    ((9, 1000), 8, None),                 # rows of odd groups
    ((2, 400, 384), 32, [400, 133]),      # columns
    ((2, 1000, 30), 2, [1000, 999]),      # columns of odd groups
    ((2, 257, 1000), 8, [257, 256]),      # splits
    ((2, 1500, 96), 1, [1500, 0]),
]


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("activation", ["relu", "silu"])
@pytest.mark.parametrize("shape,groups,lengths", SHAPES)
def test_another_output_type(shape, groups, lengths, activation, dtype, out_dtype):
    _check(shape, groups, lengths, activation, dtype, out_dtype)


def test_under_autocast():
    for shape, groups, lengths in SHAPES[:1] + SHAPES[2:3]:
        _check(shape, groups, lengths, "silu", torch.bfloat16, torch.float32, autocast=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", ["relu", "silu"])
@pytest.mark.parametrize("shape,groups", [
    ((5001, 1000), 8),   # a row a workgroup (125 channels a group, a thread each): 4096 at most forward, 1024 backward
    ((9001, 384), 6),    # two rows a workgroup or more
])
def test_more_rows_than_workgroups(shape, groups, activation, dtype):
    _check(shape, groups, None, activation, dtype, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((700, 384), 6), ((9, 1000), 8), ((3, 400, 384), 32), ((2, 2999, 384), 8)])
def test_the_backward_in_place(shape, groups, dtype):
    """dx over x, and over dy of the same dtype."""
    from asr_amd import _lib
    from asr_amd.groupnorm import group_norm_train

    dev = _dev()
    x, w, b, dy = (t.to(dev) for t in _make(shape, dtype, 3))
    dy = dy.to(dtype)
    N, T, C = shape if len(shape) == 3 else (shape[0], 1, shape[1])
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    ref = torch.autograd.grad(group_norm_train(leaves[0], groups, *leaves[1:], 1e-5, "silu"), leaves, dy)
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}[dtype]
    n = _lib.lib.lmufft_group_norm_workspace_bytes(N, T, C, groups, 1)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    m = _lib.lib.lmufft_group_norm_workspace_bytes(N, T, C, groups, 0)
    ws2 = torch.empty(max(m, 16), dtype=torch.uint8, device=dev)
    stats = torch.empty(N, groups, 2, dtype=torch.float64, device=dev)
    y = torch.empty_like(x)
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.lmufft_group_norm(x.data_ptr(), code, w.data_ptr(), b.data_ptr(), None, N, T, C, groups, 1e-5, 2, y.data_ptr(), code,
                                      stats.data_ptr(), ws2.data_ptr(), m, stream) == 0, _lib.lib.lmufft_last_error()
    for over in ("x", "dy"):
        xx, dd = x.clone(), dy.clone()
        dx = xx if over == "x" else dd
        dw, db = torch.empty_like(w), torch.empty_like(b)
        rc = _lib.lib.lmufft_group_norm_bwd(xx.data_ptr(), code, dd.data_ptr(), code, w.data_ptr(), b.data_ptr(), None, stats.data_ptr(),
                                            N, T, C, groups, 1e-5, 2, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), n, stream)
        assert rc == 0, _lib.lib.lmufft_last_error()
        for got, r in zip((dx, dw, db), ref):
            assert torch.equal(got, r), over
