"""GPU tests of the causal decay attention (k_decay, k_decay_states, k_decay_step) against the 64-bit oracle.

Tolerances, from the arithmetic.  With M the operator applied to the absolute values of its operands (the sum of the
magnitudes of all terms of an output), every term passes through at most dk products of the score, C + dk of the
contraction with v or the state, one multiplication a chunk for the state's decay and a handful for scales and powers:
    32 bits:  |err| <= (2 dk + 64 + 2 chunks + 100) 2^-24 M        (100: the exponents of the powers, off by up to
                                                                    n |log2 lambda| 2^-24 while lambda^n > e^-40)
    bf16:     + 2^-8 M (the scores, or the state, rounded once to bf16: half a step each) + 2^-8 |ref| (the output)
For random signs the roundings add in quadrature: the 2-norm of the error is held to sqrt(2) 2^-8 of the result's.
The state is held in 32 bits for both types (bf16 operands enter it in three terms): the first bound, with its own M."""
import math

import pytest
import torch

from oracle import decay_oracle as do

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a GPU")
    return torch.device("cuda:0")


def _decays(H, seed=0):
    """Slow ones as in use, and the ends of the range: everything kept, nothing kept, and nearly nothing."""
    d = [math.log1p(-2.0 ** (-5 - h % 8)) for h in range(H)]
    for h, x in ((1, 0.0), (2, -float("inf")), (3, -9.0), (4, -0.7)):
        if h < H:
            d[(h + seed) % H] = x
    return torch.tensor(d, dtype=torch.float32)


def _bound32(M, T, dk):
    return (2 * dk + 64 + 2 * (T // 32 + 1) + 100) * 2.0 ** -24 * M + 1e-30


def _close(got, ref, M, T, dk, dtype, name):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), name
    tol = _bound32(M, T, dk)
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (M + ref.abs())
        norm = float((got - ref).norm() / ref.norm().clamp(min=1e-30))
        assert norm <= 2 ** 0.5 * 2.0 ** -8 or ref.numel() < 4096, (name, norm)
    err = (got - ref).abs()
    bad = (err > tol).nonzero()
    assert len(bad) == 0, f"{name}: {len(bad)} off, first at {bad[0].tolist()}: {float(err[tuple(bad[0])]):.3e}"


def _make(B, T, H, dk, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda d: torch.randn(B, T, H * d, generator=g).to(dtype)  # noqa: E731
    return mk(dk), mk(dk), mk(dv), mk(dv), torch.randn(B, H, dk, dv, generator=g) * 3


SHAPES = [
    # B, T, H, dk, dv, lengths
    (1, 1, 1, 64, 64, None),
    (3, 2, 2, 32, 32, [2, 1, 0]),
    (2, 15, 3, 64, 32, [15, 7]),
    (2, 16, 2, 32, 64, None),
    (2, 17, 5, 64, 64, [17, 16]),
    (2, 31, 1, 128, 64, [31, 0]),
    (2, 33, 2, 64, 128, [33, 32]),
    (2, 63, 2, 128, 128, [63, 49]),
    (2, 64, 3, 64, 64, None),
    (3, 65, 2, 32, 128, [65, 64, 1]),
    (2, 127, 2, 128, 32, [127, 65]),
    (2, 129, 5, 64, 64, [129, 128]),
    (1, 400, 6, 64, 64, [317]),
    (2, 1001, 5, 64, 64, [1001, 640]),     # several segments, one utterance ends on a segment's edge
    (1, 700, 1, 128, 128, None),
    (3, 520, 2, 32, 32, [520, 0, 257]),
    (200, 70, 6, 32, 32, None),            # more heads than the chip holds at once
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,dk,dv,lengths", SHAPES)
def test_forward_with_and_without_a_state(B, T, H, dk, dv, lengths, dtype):
    from asr_amd.decay import decay_attention

    dev = _dev()
    q, k, v, _, st = _make(B, T, H, dk, dv, dtype, T)
    ld = _decays(H, T)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    args = [t.to(dev) for t in (q, k, v)]
    ref, _ = do.decay_attention(q, k, v, ld, lengths)
    M, _ = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, lengths)
    out = decay_attention(*args, H, ld.to(dev), ln)
    _close(out, ref, M, T, dk, dtype, "out")
    assert out.dtype == dtype and torch.equal(out, decay_attention(*args, H, ld.to(dev), ln))
    sd = st.to(dev)
    out = decay_attention(*args, H, ld.to(dev), ln, sd, 0.3)
    ref, S = do.decay_attention(q, k, v, ld, lengths, st, 0.3)
    M, MS = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, lengths, st.abs(), 0.3)
    _close(out, ref, M, T, dk, dtype, "out from a state")
    _close(sd, S, MS, T, 0, torch.float32, "state")
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert (out[b, n:] == 0).all()
            if n == 0:
                assert torch.equal(sd[b].cpu(), st[b])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,H,dk,dv,lengths", SHAPES)
def test_gradients(B, T, H, dk, dv, lengths, dtype):
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    q, k, v, w, _ = _make(B, T, H, dk, dv, dtype, T + 1)
    ld = _decays(H, T)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = decay_attention_train(*leaves, H, ld.to(dev), ln)
    grads = torch.autograd.grad(out, leaves, w.to(dev))
    assert torch.equal(out.detach(), decay_attention(*leaves, H, ld.to(dev), ln))
    ref = do.decay_attention_backward(q, k, v, w, ld, lengths)
    M = do.decay_attention_backward(q.abs(), k.abs(), v.abs(), w.abs(), ld, lengths)
    for got, r, m, name in zip(grads, ref, M, ("dq", "dk", "dv")):
        _close(got, r, m, T, max(dk, dv), dtype, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 64, 64), (5, 6, 64, 64), (3, 2, 32, 128), (4, 5, 128, 32), (2, 3, 128, 128)])
def test_step(B, H, dk, dv, dtype):
    from asr_amd.decay import decay_attention, decay_attention_step

    dev = _dev()
    q, k, v, _, st = _make(B, 1, H, dk, dv, dtype, 7)
    ld = _decays(H)
    active = [1 if b != 1 else 0 for b in range(B)]
    ref, S = do.decay_attention(q, k, v, ld, active, st)
    M, MS = do.decay_attention(q.abs(), k.abs(), v.abs(), ld, active, st.abs())
    for dt in (torch.int32, torch.bool):
        sd = st.to(dev)
        out = decay_attention_step(*(t[:, 0].to(dev) for t in (q, k, v)), H, ld.to(dev), sd, torch.tensor(active, device=dev).to(dt))
        _close(out, ref[:, 0], M[:, 0], 1, dk, torch.float32 if dtype == torch.float32 else dtype, "out")
        _close(sd, S, MS, 1, 0, torch.float32, "state")
        if B > 1:
            assert torch.equal(sd[1].cpu(), st[1]) and (out[1] == 0).all()
    # and the chunk form with one frame is the same operator
    sd2 = st.to(dev)
    out2 = decay_attention(*(t.to(dev) for t in (q, k, v)), H, ld.to(dev), torch.tensor(active, device=dev), sd2)
    _close(out2, ref, M, 1, dk, dtype, "chunk form")
    _close(sd2, S, MS, 1, 0, torch.float32, "its state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chunks_and_single_frames_continue_one_utterance(dtype):
    from asr_amd.decay import decay_attention, decay_attention_step

    dev = _dev()
    B, T, H, d = 2, 150, 5, 64
    q, k, v, _, _ = _make(B, T, H, d, d, dtype, 3)
    ld = _decays(H)
    ref, S = do.decay_attention(q, k, v, ld)
    M, MS = do.decay_attention(q.abs(), k.abs(), v.abs(), ld)
    a = [t.to(dev) for t in (q, k, v)]
    st = torch.zeros(B, H, d, d, device=dev)
    parts, t = [], 0
    for n in (1, 40, 1, 1, 64, 43):
        piece = [x[:, t:t + n] for x in a]  # strided views
        if n == 1:
            parts.append(decay_attention_step(*(x[:, 0] for x in piece), H, ld.to(dev), st)[:, None])
        else:
            parts.append(decay_attention(*piece, H, ld.to(dev), None, st))
        t += n
    assert t == T
    _close(torch.cat(parts, 1), ref, M, T, d, dtype, "pieces")
    _close(st, S, MS, T, 0, torch.float32, "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_and_strided_forms_are_the_same_computation(dtype):
    from asr_amd.decay import decay_attention, decay_attention_train, decay_attention_train_packed

    dev = _dev()
    B, T, H, d = 3, 130, 6, 64
    C = H * d
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(B, T, 3 * C, generator=g).to(dtype).to(dev)
    w = torch.randn(B, T, C, generator=g).to(dtype).to(dev)
    ld, ln = _decays(H).to(dev), torch.tensor([130, 64, 9], device=dev)
    a = qkv.clone().requires_grad_(True)
    out = decay_attention_train_packed(a, H, ld, ln)
    out.backward(w)
    blocks = [qkv[..., i * C:(i + 1) * C].clone().requires_grad_(True) for i in range(3)]
    ref = decay_attention_train(*blocks, H, ld, ln)
    ref.backward(w)
    assert torch.equal(out, ref) and a.grad.shape == qkv.shape
    for i, t in enumerate(blocks):
        assert torch.equal(a.grad[..., i * C:(i + 1) * C], t.grad)
    assert torch.equal(ref, decay_attention(*qkv.chunk(3, -1), H, ld, ln))                       # column blocks in place
    t_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in qkv.chunk(3, -1)]         # frames first in memory
    assert torch.equal(ref, decay_attention(*t_first, H, ld, ln))
    odd = [torch.cat([x.new_zeros(B, T, 1), x], -1)[..., 1:] for x in qkv.chunk(3, -1)]           # rows off their alignment
    assert torch.equal(ref, decay_attention(*odd, H, ld, ln))
    # one k for the whole batch, its gradient summed over it
    kk = qkv[:1, :, C:2 * C].clone().requires_grad_(True)
    out = decay_attention_train(qkv[..., :C], kk.expand(B, T, C), qkv[..., 2 * C:], H, ld, ln)
    out.backward(w)
    each = qkv[:1, :, C:2 * C].repeat(B, 1, 1).requires_grad_(True)
    decay_attention_train(qkv[..., :C], each, qkv[..., 2 * C:], H, ld, ln).backward(w)
    # a sum of three rounded values: half a step of each intermediate and of the result
    tol = torch.finfo(dtype).eps * each.grad.float().abs().sum(0, keepdim=True) + 1e-30
    assert ((kk.grad.float() - each.grad.float().sum(0, keepdim=True)).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_padding_is_not_read(dtype, poison):
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    B, T, H, d = 3, 300, 2, 64
    q, k, v, w, st = (t.to(dev) for t in _make(B, T, H, d, d, dtype, 11))
    lengths = [300, 129, 0]
    ln, ld = torch.tensor(lengths, device=dev), _decays(H).to(dev)
    bad = [t.clone() for t in (q, k, v, w)]
    for t in bad:
        for b, n in enumerate(lengths):
            t[b, n:] = poison
    s1, s2 = st.clone(), st.clone()
    assert torch.equal(decay_attention(q, k, v, H, ld, ln, s1), decay_attention(*bad[:3], H, ld, ln, s2)) and torch.equal(s1, s2)
    leaves = [t.requires_grad_(True) for t in bad[:3]]
    got = torch.autograd.grad(decay_attention_train(*leaves, H, ld, ln), leaves, bad[3])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    ref = torch.autograd.grad(decay_attention_train(*leaves, H, ld, ln), leaves, w)
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
        for i, n in enumerate(lengths):
            assert (a[i, n:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,dv,at", [(64, 64, 70), (64, 64, 64), (64, 64, 95), (32, 128, 17), (128, 128, 40), (128, 32, 127)])
def test_nothing_reaches_an_earlier_frame(d, dv, at, poison, dtype):
    """An infinity or a NaN inside the length: the frames before it come out bit for bit as without it (and so do the other
    columns behind it, where it sits in v); gradients run the other way, from an odd dout to no later frame."""
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    B, T, H = 2, 200, 2
    q, k, v, w, _ = (t.to(dev) for t in _make(B, T, H, d, dv, dtype, 19))
    ld = torch.tensor([-0.01, -0.3], device=dev)
    clean = decay_attention(q, k, v, H, ld)
    for which in range(3):
        bad = [q.clone(), k.clone(), v.clone()]
        bad[which][1, at, 5] = poison
        out = decay_attention(*bad, H, ld)
        assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :at], clean[1, :at])
        assert torch.equal(out[1, :, dv:], clean[1, :, dv:])  # the other head
        if which == 0:
            assert torch.equal(out[1, at + 1:], clean[1, at + 1:]) and not torch.isfinite(out[1, at, :dv]).any()
        elif which == 1:
            assert not torch.isfinite(out[1, at:, :dv]).any()
        else:
            assert not torch.isfinite(out[1, at:, 5]).any()
            keep = [c for c in range(dv) if c != 5]
            assert torch.equal(out[1][:, keep], clean[1][:, keep])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    ref = torch.autograd.grad(decay_attention_train(*leaves, H, ld), leaves, w)
    odd = w.clone()
    odd[1, at, 5] = poison
    got = torch.autograd.grad(decay_attention_train(*leaves, H, ld), leaves, odd)
    for a, r, name in zip(got, ref, ("dq", "dk", "dv")):
        assert torch.equal(a[0], r[0]), name
        after = slice(at + 1, T) if name != "dq" else [t for t in range(T) if t != at]
        assert torch.equal(a[1, after], r[1, after]), name


@pytest.mark.parametrize("T,H,d,dv", [(1, 2, 64, 64), (3, 12, 64, 64), (17, 2, 32, 128), (32, 3, 128, 128), (64, 1, 64, 32)])
def test_few_frames_lose_only_the_outputs_rounding(T, H, d, dv):
    """Calls of one chunk in bf16: P in two bf16 terms (2^-9 each, 2^-16 M with room), the rest as in 32 bits, and half a step of
    the result."""
    from asr_amd.decay import decay_attention_train

    dev = _dev()
    q, k, v, w, _ = _make(2, T, H, d, dv, torch.bfloat16, 23)
    w, ld = w.to(torch.bfloat16), _decays(H)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = decay_attention_train(*leaves, H, ld.to(dev))
    got = [out.detach(), *torch.autograd.grad(out, leaves, w.to(dev))]
    args = [t.double() for t in (q, k, v, w)]
    size = [t.abs() for t in args]
    ref = [do.decay_attention(*args[:3], ld.double())[0], *do.decay_attention_backward(*args, ld.double())]
    M = [do.decay_attention(*size[:3], ld.double())[0], *do.decay_attention_backward(*size, ld.double())]
    for name, g, r, m in zip(("out", "dq", "dk", "dv"), got, ref, M):
        err = (g.double().cpu() - r).abs()
        assert (err <= _bound32(m, T, max(d, dv)) + 2.0 ** -16 * m + 2.0 ** -8 * r.abs()).all(), (name, float(err.max()))


def test_rows_far_apart():
    """A transposed view whose frames lie 2^22 elements and more apart is copied, not refused."""
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    q, k, v, w, _ = (t.to(dev) for t in _make(2, 3, 2, 32, 32, torch.bfloat16, 8))
    ld = _decays(2).to(dev)
    far = torch.empty(3 * ((1 << 22) + 64), dtype=torch.bfloat16, device=dev).as_strided((2, 3, 64), (64, (1 << 22) + 64, 1))
    far.copy_(k)
    assert torch.equal(decay_attention(q, far, v, 2, ld), decay_attention(q, k, v, 2, ld))
    leaves = [q.clone().requires_grad_(True), far.detach().requires_grad_(True), v.clone().requires_grad_(True)]
    got = torch.autograd.grad(decay_attention_train(*leaves, 2, ld), leaves, w)
    leaves[1] = k.clone().requires_grad_(True)
    ref = torch.autograd.grad(decay_attention_train(*leaves, 2, ld), leaves, w)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_lengths_of_64_bits():
    from asr_amd.decay import decay_attention

    dev = _dev()
    q, k, v, _, _ = (t.to(dev) for t in _make(3, 40, 2, 32, 32, torch.float32, 6))
    ld = _decays(2).to(dev)
    ref = decay_attention(q, k, v, 2, ld, torch.tensor([40, 0, 9], dtype=torch.int32, device=dev))
    assert torch.equal(decay_attention(q, k, v, 2, ld, torch.tensor([1 << 40, -(1 << 40), 9])), ref)


def test_gradients_against_differences():
    """Along a random direction; f32, so a central difference of step h is off by h^2 / 6 of the third derivative -- zero in
    each single operand, in which the operator is linear -- and by rounding, 2^-24 of the sum's magnitudes over h."""
    from asr_amd.decay import decay_attention, decay_attention_train

    dev = _dev()
    B, T, H, d = 2, 200, 3, 32
    q, k, v, w, _ = (t.to(dev) for t in _make(B, T, H, d, d, torch.float32, 23))
    ld, ln = torch.tensor([-0.05, -0.01, 0.0], device=dev), torch.tensor([200, 77], device=dev)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(decay_attention_train(*leaves, H, ld, ln), leaves, w)
    for i in range(3):
        u = torch.randn_like(leaves[i])
        f = lambda s: (decay_attention(*[t.detach() + (s * u if j == i else 0) for j, t in enumerate(leaves)], H, ld, ln).double()  # noqa: E731
                       * w.double()).sum()
        size = decay_attention(*[t.detach().abs() + (u.abs() if j == i else 0) for j, t in enumerate(leaves)], H, ld, ln).double()
        most = 400 * 2.0 ** -24 * float((size * w.double().abs()).sum())
        assert abs(float((f(1.0) - f(-1.0)) / 2) - float((grads[i].double() * u.double()).sum())) <= most


@pytest.mark.parametrize("B,T,H,d", [(2, 700, 2, 64), (1, 300, 3, 128), (1, 1500, 1, 32)])
def test_captured_calls_replay(B, T, H, d):
    """A prompt and a step captured together, and a training pass: every replay against the eager result, with eager calls
    of the same operators in between."""
    from asr_amd.decay import decay_attention, decay_attention_step, decay_attention_train_packed

    dev = _dev()
    q, k, v, _, st = (t.to(dev) for t in _make(B, T, H, d, d, torch.bfloat16, 31))
    ld, ln = _decays(H).to(dev), torch.tensor([T, T // 2 - 17][:B], dtype=torch.int32, device=dev)
    qkv = torch.cat([q, k, v], -1).requires_grad_(True)
    w = torch.randn_like(q)

    def serve(state):
        a = decay_attention(q, k, v, H, ld, ln, state)
        return a, decay_attention_step(q[:, 0], k[:, 0], v[:, 0], H, ld, state)

    def train():
        out = decay_attention_train_packed(qkv, H, ld, ln)
        return out.detach(), *torch.autograd.grad(out, qkv, w)

    state = st.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve(state)
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = (*serve(state), *train())
    for i in range(4):
        with torch.no_grad():
            qkv.mul_(-1)
            q.mul_(0.5 if i % 2 else 2.0)
        state.copy_(st)
        graph.replay()
        torch.cuda.synchronize()
        end = st.clone()
        ref = (*serve(end), *train())
        for a, b in zip(got, ref):
            assert torch.equal(a, b), i
        assert torch.equal(state, end)


def test_another_stream_and_two_at_once():
    from asr_amd.decay import decay_attention

    dev = _dev()
    a = [t.to(dev) for t in _make(2, 900, 2, 64, 64, torch.bfloat16, 41)[:3]]
    b = [t.to(dev) for t in _make(3, 800, 1, 64, 64, torch.bfloat16, 42)[:3]]
    la, lb = _decays(2).to(dev), _decays(1).to(dev)
    ra, rb = decay_attention(*a, 2, la), decay_attention(*b, 1, lb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = decay_attention(*a, 2, la)
        with torch.cuda.stream(s2):
            y = decay_attention(*b, 1, lb)
        torch.cuda.synchronize()
        assert torch.equal(x, ra) and torch.equal(y, rb)


def test_empty_calls_and_refusals():
    from asr_amd import decay

    dev = _dev()
    x, ld = torch.zeros(2, 5, 128, device=dev), torch.zeros(2, device=dev)
    st = torch.ones(2, 2, 64, 64, device=dev)
    assert decay.decay_attention(x[:, :0], x[:, :0], x[:, :0], 2, ld, None, st).shape == (2, 0, 128) and (st == 1).all()
    assert decay.decay_attention(x[:0], x[:0], x[:0], 2, ld).shape == (0, 5, 128)
    assert decay.decay_attention_step(x[:0, 0], x[:0, 0], x[:0, 0], 2, ld, st[:0]).shape == (0, 128)
    e = x[:, :0].clone().requires_grad_(True)
    decay.decay_attention_train(e, e, e, 2, ld).sum().backward()
    assert e.grad.shape == (2, 0, 128)
    bad = [
        (dict(num_heads=3), "do not split"), (dict(num_heads=8), "head widths"), (dict(log_decay=ld[:1]), "log_decay"),
        (dict(log_decay=ld.double()), "log_decay"), (dict(log_decay=ld.cpu()), "no CPU fallback"),
        (dict(lengths=torch.ones(3, device=dev)), "lengths"), (dict(state=st[:1]), "`state`"), (dict(state=st.double()), "`state`"),
        (dict(state=st.transpose(2, 3)), "`state`"), (dict(k=x[:, :4]), "share one"), (dict(v=x[:1]), "share one"),
        (dict(log_decay=ld.clone().requires_grad_(True)), "constants"), (dict(state=st.clone().requires_grad_(True)), "gradient"),
    ]
    for change, text in bad:
        kw = dict(q=x, k=x, v=x, num_heads=2, log_decay=ld) | change
        with pytest.raises(RuntimeError, match=text):
            decay.decay_attention(**kw)
    y = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(decay.decay_attention_train(y, x, x, 2, ld).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):  # the backward has no backward of its own
        torch.autograd.grad(g.sum(), y)
