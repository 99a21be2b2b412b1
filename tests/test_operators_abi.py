"""CPU-side checks of the operators' C entry points: what they refuse before any launch."""


def test_the_group_norm_refuses_to_write_over_another_type():
    """In place with one dtype is fine; a result of another element size over its input is not (checked before any launch)."""
    from asr_amd import _lib

    lib, p = _lib.lib, 1 << 20
    for x, y in ((_lib.BF16, _lib.F32), (_lib.F32, _lib.BF16)):
        for T in (1, 10):
            rc = lib.lmufft_group_norm(p, x, 2 * p, 2 * p, None, 2, T, 64, 4, 1e-5, 0, p, y, None, 3 * p, 1 << 20, None)
            assert rc != 0 and b"alias" in lib.lmufft_last_error(), lib.lmufft_last_error()
            rc = lib.lmufft_group_norm_bwd(3 * p, x, p, y, 2 * p, 2 * p, None, 4 * p, 2, T, 64, 4, 1e-5, 0, p, 5 * p, 5 * p + 1024,
                                           6 * p, 1 << 20, None)
            assert rc != 0 and b"alias" in lib.lmufft_last_error(), lib.lmufft_last_error()
            # a result that begins inside its input
            rc = lib.lmufft_group_norm(p, x, 2 * p, 2 * p, None, 2, T, 64, 4, 1e-5, 0, p + 64, x, None, 3 * p, 1 << 20, None)
            assert rc != 0 and b"alias" in lib.lmufft_last_error(), lib.lmufft_last_error()


def test_the_decay_attention_s_segments_follow_the_heads_without_a_jump():
    """The workspace holds a state for every segment: one head more leaves at least 0.6 of an utterance's segments (their length
    is a whole number of chunks, two or more, which alone may leave two thirds)."""
    from asr_amd import _lib

    def segments(dtype, T, heads, d):
        return max(1, _lib.lib.lmufft_decay_workspace_bytes(dtype, 1, T, heads, d, d, 0) // (4 * heads * d * d))

    for dtype in (_lib.F32, _lib.BF16):
        for d in (32, 64, 128):
            for T in (400, 3000, 8000, 24000):
                n = [segments(dtype, T, h, d) for h in range(1, 161)]
                assert n[0] > 1 and all(a >= b for a, b in zip(n, n[1:])), (dtype, d, T)
                assert all(b >= 0.6 * a or a == 2 for a, b in zip(n, n[1:])), (dtype, d, T, n)
