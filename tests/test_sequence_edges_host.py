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
