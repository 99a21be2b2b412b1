"""GPU tests of the group norm with an activation (k_gn_rows, k_gn_stats, k_gn_apply and their backwards) against the
64-bit oracle.

Tolerances, from the arithmetic, u = 2^-24, E = 160 + T + N a bound of the roundings a sum's terms pass through (a thread's
own additions, the trees, the partials) and of the few around them.  A group's mean is off by at most E u A (A: the largest
|x| of its group), so |d xhat| <= h = E u (|xhat| + A rstd), and with slopes of at most 1.1 and curvatures of at most 0.5:
    |dy err|  <= 1.1 |w| h + (2 |z| + 20) u (|z| + |b|)          (the exponential's argument carries |z| u)
    |dx err|  <= rstd (E u (|g| + m|g| + |xhat| m|g xhat|) + h (|m(g xhat)| + |dy w|) + m(|dy w| h) (1 + |xhat|)) + (2|z|+20) u |dy w| rstd
    |dw err|  <= sum E u |dz xhat| + |dz| h + |dy xhat| (0.5 |w| h + (2 |z| + 20) u),   |db err| the same without xhat
(g = dz w, m = mean over the group.)  A bf16 result adds half a step, 2^-8 |ref|.  The ReLU's slope jumps at zero: where |z|
is within 1e-4 of it the incoming gradient is zero, so that no side is asked which way it rounds."""
import pytest
import torch

from oracle import groupnorm_oracle as go

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _dev():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a GPU")
    return torch.device("cuda:0")


def _make(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=g) * (0.3 + torch.rand(C, generator=g)) + 2 * torch.randn(C, generator=g)).to(dtype)
    return x, 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g), torch.randn(*shape, generator=g)


def _pieces(x, G, w, b, lengths):
    """xhat, rstd, z, A and a group-mean function, broadcast to x's shape (samples behind their length: zeros)."""
    hat, rstd, A = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    parts = go._parts(x, lengths)
    for at, part in parts:
        h, r = go._normalised(part, G, 1e-5)
        hat[at] = h.reshape(hat[at].shape)
        rstd[at] = r.expand_as(h).reshape(hat[at].shape)
        p = part.abs().reshape(part.shape[0], G, -1)
        A[at] = p.amax(dim=(0, 2), keepdim=True).expand_as(p).reshape(hat[at].shape)

    def mean(t):
        m = torch.zeros_like(t)
        for at, part in parts:
            p = t[at].reshape(part.shape[0], G, -1)
            m[at] = p.mean(dim=(0, 2), keepdim=True).expand_as(p).reshape(m[at].shape)
        return m

    return hat, rstd, hat * w + b, A, mean


def _within(got, ref, tol, dtype, name):
    got = got.detach().double().cpu()
    if dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()
    err = (got - ref).abs()
    bad = (~(err <= tol + 1e-30)).nonzero()
    assert len(bad) == 0, f"{name}: {len(bad)} off, first at {bad[0].tolist()}: {float(err[tuple(bad[0])]):.3e}"


CASES = [
    # shape, groups, lengths
    ((1, 64), 1, None),
    ((7, 384), 6, None),
    ((501, 384), 32, None),          # twelve channels a group: three vectors of four
    ((33, 80), 5, None),
    ((9, 1000), 8, None),            # odd groups: 125 channels
    ((40, 1000), 1, None),
    ((3, 6), 6, None),               # one channel a group: its own mean
    ((2500, 128), 2, None),
    ((6000, 16), 1, None),
    ((1, 1, 64), 4, None),
    ((3, 1, 96), 4, [1, 0, 1]),
    ((2, 2, 96), 96, [2, 1]),
    ((3, 17, 384), 6, [17, 9, 0]),
    ((2, 400, 384), 32, [400, 133]),
    ((1, 1000, 80), 5, None),
    ((2, 257, 1000), 8, [257, 256]),
    ((4, 130, 250), 2, [130, 129, 2, 1]),
    ((70, 50, 64), 1, None),
    # odd groups of long utterances: as many frames a thread as the kernels keep, and more than that
    ((2, 1000, 30), 2, [1000, 999]),
    ((1, 700, 18), 2, None),
    ((3, 680, 30), 2, [680, 1, 341]),
    ((2, 1100, 30), 2, None),
    ((110, 500, 10), 5, None),
    ((2, 2600, 12), 2, [2600, 2599]),
    ((200, 170, 36), 3, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", [None, "relu", "silu"])
@pytest.mark.parametrize("shape,groups,lengths", CASES)
def test_forward_and_backward(shape, groups, lengths, activation, dtype):
    from asr_amd.groupnorm import group_norm, group_norm_train

    dev = _dev()
    x, w, b, dy = _make(shape, dtype, shape[0] * 7 + groups)
    xd = x.double()
    hat, rstd, z, A, mean = _pieces(xd, groups, w.double(), b.double(), lengths)
    if activation == "relu":
        dy = torch.where(z.abs() < 1e-4, 0.0, dy.double()).float()
    dy = dy.to(dtype)
    ln = None if lengths is None else torch.tensor(lengths, device=dev)
    leaves = [x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)]
    y = group_norm_train(leaves[0], groups, *leaves[1:], 1e-5, activation, ln)
    grads = torch.autograd.grad(y, leaves, dy.to(dev))
    again = group_norm(leaves[0], groups, *leaves[1:], 1e-5, activation, ln)
    assert y.dtype == dtype and torch.equal(y, again)

    E = 160 + (shape[1] if len(shape) == 3 else 1) + shape[0]
    w, b, dyd = w.double(), b.double(), dy.double()
    h = E * U * (hat.abs() + A * rstd)
    soft = (2 * z.abs() + 20) * U
    ref = go.group_norm(x, groups, w, b, 1e-5, activation, lengths)
    _within(y, ref, 1.1 * w.abs() * h + soft * (z.abs() + b.abs()), dtype, "y")
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
    if lengths is not None:
        for i, n in enumerate(lengths):
            assert (y[i, n:] == 0).all() and (grads[0][i, n:] == 0).all()


def test_large_offsets_keep_their_variance():
    """x = 1000 + noise: a variance from sums of squares would be lost; about a value of the data it is not.  The rounding of
    x - mean is exact here (neighbouring values), so only the mean's own rounding, 2^-24 1000, shifts xhat."""
    from asr_amd.groupnorm import group_norm

    dev = _dev()
    g = torch.Generator().manual_seed(2)
    for shape in ((64, 96), (2, 500, 96)):
        x = 1000 + torch.randn(*shape, generator=g)
        w, b = torch.ones(96), torch.zeros(96)
        ref = go.group_norm(x, 4, w, b)
        got = group_norm(x.to(dev), 4, w.to(dev), b.to(dev)).double().cpu()
        sums = 30 if len(shape) == 2 else 4  # roundings of a sum of 24 values near 1000; the utterances' means are joined in 64 bits
        assert float((got - ref).abs().max()) <= 1000 * U * sums * 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((200, 384), 6), ((300, 60), 4), ((3, 400, 384), 32), ((2, 3000, 96), 2)])
def test_the_border_of_the_relu_is_decided_exactly(shape, groups, dtype):
    """Biases that put one element of each channel within a rounding of zero (2^-25 of the bias, far inside what 32 bits can
    tell): its slope is the sign's all the same.  The statistics are exact to 64 bits; every such z is above 1e-13."""
    from asr_amd.groupnorm import group_norm_train

    dev = _dev()
    C = shape[-1]
    x, w, _, _ = _make(shape, dtype, 77)
    hat, *_ = _pieces(x.double(), groups, w.double(), torch.zeros(C, dtype=torch.float64), None)
    g = torch.Generator().manual_seed(5)
    rows = hat.reshape(-1, C)
    at = torch.randint(0, rows.shape[0], (C,), generator=g)
    cols = torch.arange(C)
    b = (-rows[at, cols] * w.double()).float()
    z = rows[at, cols] * w.double() + b.double()
    assert (z.abs() > 1e-13).all() and (z.abs() < 1e-6).all() and 0.2 < float((z > 0).double().mean()) < 0.8
    dy = torch.zeros(rows.shape)
    dy[at, cols] = 1.0
    leaves = [x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True), b.to(dev).requires_grad_(True)]
    y = group_norm_train(leaves[0], groups, *leaves[1:], 1e-5, "relu")
    dx, dw, db = torch.autograd.grad(y, leaves, dy.reshape(shape).to(dtype).to(dev))
    assert torch.equal(db.cpu(), (z > 0).float())
    rx, rw, _ = go.group_norm_backward(x, groups, w, b, dy.reshape(shape), 1e-5, "relu")
    assert ((dw.double().cpu() - rw).abs() <= 200 * U * rw.abs() + 200 * U * 8).all()  # (one term a channel; |xhat| below 8)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_padding_is_not_read(poison):
    from asr_amd.groupnorm import group_norm_train

    dev = _dev()
    lengths = [90, 31, 0]
    ln = torch.tensor(lengths, device=dev)
    x, w, b, dy = (t.to(dev) for t in _make((3, 90, 96), torch.float32, 5))
    bad, bad_dy = x.clone(), dy.clone()
    for i, n in enumerate(lengths):
        bad[i, n:] = poison
        bad_dy[i, n:] = poison
    res = []
    for xx, dd in ((x, dy), (bad, bad_dy)):
        leaves = [t.clone().requires_grad_(True) for t in (xx, w, b)]
        y = group_norm_train(leaves[0], 4, *leaves[1:], 1e-5, "silu", ln)
        res.append((y.detach(), *torch.autograd.grad(y, leaves, dd)))
    for a, r in zip(*res):
        assert torch.equal(a, r) and torch.isfinite(a).all()


def test_output_types_layouts_and_parameters():
    from asr_amd.groupnorm import group_norm, group_norm_train
    from asr_amd.parallel import GradBuckets

    dev = _dev()
    x, w, b, dy = (t.to(dev) for t in _make((3, 40, 96), torch.bfloat16, 8))
    y32 = group_norm(x, 4, w, b, out_dtype=torch.float32)
    assert y32.dtype == torch.float32 and torch.equal(y32.bfloat16(), group_norm(x, 4, w, b))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert group_norm(x, 4, w, b).dtype == torch.float32
    assert torch.equal(group_norm(x.transpose(0, 1).contiguous().transpose(0, 1), 4, w, b), group_norm(x, 4, w, b))
    wide = torch.cat([x.new_zeros(3, 40, 1), x], -1)[..., 1:]
    assert torch.equal(group_norm(wide, 4, w, b), group_norm(x, 4, w, b))
    assert torch.equal(group_norm(x, 4, w.bfloat16(), b.bfloat16()), group_norm(x, 4, w.bfloat16().float(), b.bfloat16().float()))
    # parameters of a gradient bucket: written in place
    pw, pb = torch.nn.Parameter(w.clone()), torch.nn.Parameter(b.clone())
    buckets = GradBuckets([[pw, pb]], overlap=False)
    buckets.zero_grad()
    group_norm_train(x, 4, pw, pb, 1e-5, "silu").backward(dy.to(torch.bfloat16))
    buckets.finish()
    lw, lb = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    group_norm_train(x, 4, lw, lb, 1e-5, "silu").backward(dy.to(torch.bfloat16))
    assert torch.equal(pw.grad, lw.grad) and torch.equal(pb.grad, lb.grad)
    # used twice in one step: the gradients add up
    buckets.zero_grad()
    (group_norm_train(x, 4, pw, pb, 1e-5, "silu").float() + group_norm_train(x, 4, pw, pb, 1e-5, "silu").float()).backward(dy)
    buckets.finish()
    l2w, l2b = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    group_norm_train(x, 4, l2w, l2b, 1e-5, "silu").backward(dy.to(torch.bfloat16))
    tol = 4 * U * l2w.grad.abs() + 4 * U
    assert ((pw.grad - 2 * l2w.grad).abs() <= tol).all()
    buckets.remove()


def test_captured_training_pass_replays():
    from asr_amd.groupnorm import group_norm_train

    dev = _dev()
    x, w, b, dy = (t.to(dev) for t in _make((3, 400, 384), torch.float32, 9))
    rows = x[0].clone().requires_grad_(True)
    ln = torch.tensor([400, 17, 0], dtype=torch.int32, device=dev)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def go_():
        y = group_norm_train(x, 32, w, b, 1e-5, "silu", ln)
        r = group_norm_train(rows, 6, w, b, 1e-5, "relu")
        return (y.detach(), r.detach(), *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(r, (rows, w, b), dy[0]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go_()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go_()
    for i in range(4):
        with torch.no_grad():
            x.mul_(-1.5)
            rows.add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(got, go_()):
            assert torch.equal(a, r), i


@pytest.mark.parametrize("shape,groups", [((3, 2999, 384), 8), ((2, 5000, 96), 3), ((4, 100, 96), 4), ((500, 1, 384), 6)])
def test_in_place(shape, groups):
    """out == x of one dtype: what the result is made of is read before anything is written over it."""
    from asr_amd import _lib
    from asr_amd.groupnorm import group_norm

    dev = _dev()
    N, T, C = shape
    x, w, b, _ = (t.to(dev) for t in _make(shape, torch.float32, 12))
    lengths = torch.tensor([T, T // 2, 0, 1][:N], dtype=torch.int32, device=dev) if T > 1 else None
    ref = group_norm(x, groups, w, b, activation="silu", lengths=lengths)
    n = _lib.lib.lmufft_group_norm_workspace_bytes(N, T, C, groups, 0)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=dev)
    for _ in range(20):
        y = x.clone()
        rc = _lib.lib.lmufft_group_norm(y.data_ptr(), _lib.F32, w.data_ptr(), b.data_ptr(), None if lengths is None else lengths.data_ptr(),
                                        N, T, C, groups, 1e-5, 2, y.data_ptr(), _lib.F32, None, ws.data_ptr(), n,
                                        torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.lib.lmufft_last_error()
        assert torch.equal(y, ref)


def test_lengths_of_64_bits():
    from asr_amd.groupnorm import group_norm

    dev = _dev()
    x, w, b, _ = (t.to(dev) for t in _make((3, 20, 96), torch.float32, 4))
    ref = group_norm(x, 4, w, b, lengths=torch.tensor([20, 0, 7], dtype=torch.int32, device=dev))
    assert torch.equal(group_norm(x, 4, w, b, lengths=torch.tensor([1 << 40, -(1 << 40), 7])), ref)


def test_empty_calls_and_refusals():
    from asr_amd.groupnorm import group_norm, group_norm_train

    dev = _dev()
    w = torch.ones(96, device=dev, requires_grad=True)
    for shape in ((0, 5, 96), (2, 0, 96), (0, 96)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        y = group_norm_train(x, 4, w, w, 1e-5, "silu")
        y.sum().backward()
        assert y.shape == shape and x.grad.shape == shape and (w.grad == 0).all()
        w.grad = None
    x = torch.zeros(2, 5, 96, device=dev)
    with pytest.raises(RuntimeError, match="weight and bias"):
        group_norm(x, 4, w[:95], w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_norm(x, 4, w.cpu(), w)
    with pytest.raises(RuntimeError, match="lengths"):
        group_norm(x, 4, w, w, lengths=torch.ones(3, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="lengths go with"):
        group_norm(x[0], 4, w, w, lengths=torch.ones(5, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="whole numbers"):
        group_norm(x, 4, w, w, lengths=torch.ones(2, device=dev))
    assert (group_norm(x, 4, w, torch.full((96,), -1.0, device=dev), activation="relu") == 0).all()  # a constant sample
    y = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(group_norm_train(y, 4, w, w).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):  # the backward has no backward of its own
        torch.autograd.grad(g.sum(), y)
