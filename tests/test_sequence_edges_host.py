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
