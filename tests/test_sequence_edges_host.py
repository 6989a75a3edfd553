"""Host side of the token-sequence operators, further refusals (no GPU needed)."""
import pytest
import torch


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def test_calls_without_key_heads_are_refused():
    """Pages of no key head leave nothing to launch over: the results would be memory nobody wrote."""
    from aot_hip import AotHipError
    from networks.layers import sequence as S
    q, none, kp = torch.zeros(5, 4, 32), torch.zeros(5, 0, 32), torch.zeros(6, 8, 0, 32)
    with pytest.raises(AotHipError, match='at least one key head'):
        S.rope_append(q, none, none, i32(5), S.rope_freqs(32), i32(5), kp, kp)
    with pytest.raises(AotHipError, match='at least one key head'):
        S.paged_evict(kp, kp, i32(2, 3), i32(2), torch.zeros(2, 0, 24), i32(2, 1), 8)


def test_frequencies_that_want_a_gradient_are_refused():
    """rope is differentiable in q and k only: a gradient of the frequencies is refused, as one of the slopes is, and not returned as none."""
    from aot_hip import AotHipError
    from networks.layers import sequence as S
    q, k, pos, f = torch.zeros(1, 4, 4, 32), torch.zeros(1, 4, 2, 32), i32(1, 4), S.rope_freqs(32).requires_grad_()
    kp = torch.zeros(6, 8, 2, 32)
    for other in (k, None):
        with pytest.raises(AotHipError, match='freqs have no gradient'):
            S.rope(q, other, pos, f)
        with torch.no_grad(), pytest.raises(AotHipError, match='no CPU fallback'):     # nothing asks for one: as any call
            S.rope(q, other, pos, f)
    with pytest.raises(AotHipError, match='serving call'):
        S.rope_append(q[0], k[0], k[0], pos[0], f, pos[0], kp, kp)


def test_sizes_past_the_kernels_index_range_are_refused():
    """Eviction counts a row's entries and the waves' runs of them in 32 bits: 2^30 entries a row, as in paged attention.  A launch's work
    items are below 2^32 a dimension, which is looked at before anything is launched."""
    import ctypes
    import aot_hip
    from networks.layers import sequence as S
    lib, P = aot_hip.load(), ctypes.c_void_p
    z14, z16 = (ctypes.c_long * 14)(), (ctypes.c_long * 16)()

    def evict(page=1 << 16, mp=1, npg=1, budget=16):
        return lib.aot_paged_evict(P(16), P(16), P(16), P(32), P(16), P(16), None, P(16), P(32), P(32), None, 1, 1, 1, 32, mp * page, page, mp, npg, 9, budget,
                                   1, 1, z16, None)
    assert evict(mp=(1 << 14) + 1) == -2 and evict(npg=(1 << 14) + 1) == -2 and evict(npg=1 << 14, budget=1 << 29) == -2
    page, i = torch.zeros(1, 1 << 10, 2, 32), i32(1)
    with pytest.raises(aot_hip.AotHipError, match='beyond'):
        S.paged_evict(page, page, i32(1, (1 << 20) + 1), i, torch.zeros(1).expand(1, 2, (1 << 30) + (1 << 10)), i32(1, 1), 8)
    with pytest.raises(aot_hip.AotHipError, match='beyond'):
        S.paged_evict(page, page, i32(1, 1), i, torch.zeros(1, 2, 1 << 10), i32(1, (1 << 20) + 1), 8)
    assert lib.aot_rope(P(16), None, P(16), None, P(16), P(16), 0, 1 << 13, 1 << 13, 1, 0, 32, 32, 0, 0, 1.0, z14, None) == -2      # 2^26 tokens, four a workgroup
    assert lib.aot_attn_masked(P(16), P(16), P(16), P(16), None, P(16), None, None, None, None, None, None, 0, 0, 1 << 12, 1, 1, 1 << 12, 1, 32, 0, 1.0, 0.0,
                               z14, None) == -2
