"""Host side of the token-sequence operators: what the C entries and the Python calls refuse, before any launch (no GPU needed)."""
import ctypes
import math

import pytest
import torch

import sequence_refs as R


def L(*x):
    return (ctypes.c_long * len(x))(*x)


P = ctypes.c_void_p


def test_c_entries_refuse_before_any_launch():
    import aot_hip
    lib = aot_hip.load()
    z14, z15, z16, z26 = (L(*[0] * n) for n in (14, 15, 16, 26))

    def rope(q=P(16), k=P(16), qo=P(16), ko=P(16), pos=P(16), freqs=P(16), dtype=0, B=1, S=1, H=1, Hk=1, D=32, rot=32, inter=0, st=z14):
        return lib.aot_rope(q, k, qo, ko, pos, freqs, dtype, B, S, H, Hk, D, rot, inter, 0, 1.0, st, None)
    for bad in (dict(dtype=3), dict(rot=33), dict(rot=34), dict(rot=0), dict(H=0, Hk=0), dict(H=-1), dict(B=-1), dict(pos=None), dict(q=None),
                dict(ko=None), dict(st=None), dict(inter=1, q=P(20)), dict(inter=1, D=33)):
        assert rope(**bad) == -1, bad
    assert rope(D=1026, rot=32) == -2
    assert rope(B=0) == 0 and rope(S=0, q=None, k=None) == 0

    def append(N=1, H=1, Hk=1, D=32, rot=32, page=16, pages=4, dtype=0, slots=P(16), kp=P(16)):
        return lib.aot_rope_append(P(16), P(16), P(16), P(16), kp, P(16), P(16), slots, P(16), dtype, N, H, Hk, D, rot, 0, 1.0, page, pages, z14, None)
    for bad in (dict(page=12), dict(page=0), dict(slots=None), dict(Hk=0), dict(kp=None), dict(dtype=-1), dict(N=-1)):
        assert append(**bad) == -1, bad
    assert append(pages=1 << 28) == -2 and append(N=0) == 0

    def masked(dtype=0, B=1, Sq=1, Sk=1, H=1, Hk=1, D=32, cap=0.0, q=P(16), k=P(16), dq=None, dk=None, rng=None, st=z14, lse=P(16), res=None, scale=1.0):
        return lib.aot_attn_masked(q, k, P(16), P(16), res, lse, None, dq, dk, None, rng, None, 0, dtype, B, Sq, Sk, H, Hk, D, 1, scale, cap, st, None)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(cap=math.inf), dict(dtype=7), dict(H=3, Hk=2), dict(Hk=0), dict(cap=-1.0), dict(cap=math.nan), dict(dq=P(16)), dict(dq=P(16), dk=P(16)), dict(q=P(24)), dict(q=None),
                dict(k=None), dict(lse=None), dict(st=None), dict(res=P(24)), dict(Sk=4096), dict(st=L(0, 33, *[0] * 12)), dict(Sq=-1), dict(D=0)):
        assert masked(**bad) == -1, bad
    assert masked(D=132) == -2 and masked(D=33) == -2 and masked(dtype=1, D=36) == -2 and masked(Sk=(1 << 22) + 1) == -2
    assert masked(B=0) == 0 and masked(Sq=0, q=None) == 0

    def bwd(Sq=1, Sk=1, dk=P(16), delta=P(16), do=P(16), st=z26, D=32, floats=1 << 20):
        return lib.aot_attn_masked_bwd(P(16), P(16), P(16), P(16), None, P(16), do, P(16), dk, P(16), None, None, None, None, None, delta, floats, 2, 1, Sq, Sk, 1, 1, D, 0,
                                       1.0, 0.0, st, None)
    assert bwd(floats=3) == -1 and bwd(delta=P(20)) == -1 and bwd(dk=P(24)) == -1 and bwd(dk=None) == -1 and bwd(delta=None) == -1 and bwd(do=P(18)) == -1 and bwd(st=None) == -1 and bwd(D=136) == -2
    assert bwd(Sq=0, Sk=0, dk=None) == 0

    def paged(dtype=0, B=1, H=1, Hk=1, D=32, page=16, mp=1, pages=4, cap=0.0, q=P(16), kp=P(16), work=None, floats=0, w=None, st=z15, table=P(16)):
        return lib.aot_paged_attn(q, kp, P(16), table, P(16), None, None, w, P(16), work, floats, dtype, B, H, Hk, D, page, mp, pages, 1.0, cap, st, None)
    for bad in (dict(dtype=9), dict(page=24), dict(H=3, Hk=2), dict(cap=-0.5), dict(q=P(8)), dict(kp=P(8)), dict(kp=None), dict(table=None), dict(st=None),
                dict(w=P(16)), dict(mp=4096), dict(mp=4096, work=P(16), floats=5), dict(st=L(0, 0, 0, 0, 2, *[0] * 10)), dict(mp=-1)):
        assert paged(**bad) == -1, bad
    assert paged(D=260) == -2 and paged(D=30) == -2 and paged(page=1 << 20, mp=1 << 12) == -2 and paged(B=0) == 0
    n = ctypes.c_long(-1)
    assert lib.aot_paged_attn_work_floats(1, 8, 2, 64, 16, 4, 0, ctypes.addressof(n)) == 0 and n.value == 0
    assert lib.aot_paged_attn_work_floats(1, 8, 2, 64, 16, 4, 1, ctypes.addressof(n)) == 0 and n.value >= 8 * (64 + 66)
    assert lib.aot_paged_attn_work_floats(4096, 64, 8, 64, 1 << 20, 1 << 12, 1, ctypes.addressof(n)) == -2
    assert lib.aot_paged_attn_work_floats(4096, 64, 8, 64, 1 << 20, 1 << 10, 0, ctypes.addressof(n)) == 0 and n.value == 0      # one split of 2^30
    assert lib.aot_paged_attn_work_floats(1, 8, 3, 64, 16, 4, 1, ctypes.addressof(n)) == -1
    assert lib.aot_paged_attn_work_floats(1, 8, 2, 64, 16, 4, 1, None) == -1

    def evict(dtype=1, B=1, Hk=1, D=32, S=64, page=16, mp=4, npg=1, pages=9, budget=16, sink=1, recent=1, kp=P(16), new=P(32), w=P(16), nw=P(32), pos=None,
              npos=None, st=z16):
        return lib.aot_paged_evict(kp, P(16), P(16), new, P(16), w, pos, P(16), P(32), nw, npos, dtype, B, Hk, D, S, page, mp, npg, pages, budget, sink, recent,
                                   st, None)
    for bad in (dict(dtype=5), dict(page=20), dict(budget=0), dict(budget=17), dict(sink=9, recent=8), dict(sink=-1), dict(kp=None), dict(new=P(16)), dict(nw=P(16)),
                dict(w=None), dict(pos=P(16)), dict(pos=P(16), npos=P(16)), dict(st=None), dict(Hk=0)):
        assert evict(**bad) == -1, bad
    assert evict(page=1 << 16, mp=1 << 15, budget=16) == -2 and evict(B=0) == 0


def test_python_calls_refuse_what_the_kernels_do_not_take():
    """On CPU tensors: wrong shapes and types are named first, a right call fails for want of a device."""
    from aot_hip import AotHipError
    from networks.layers import sequence as S
    f = torch.zeros
    i32 = lambda *s: f(*s, dtype=torch.int32)                                 # noqa: E731
    q, k, pos, freqs = f(1, 4, 4, 32), f(1, 4, 2, 32), i32(1, 4), S.rope_freqs(32)
    kp, table, n, w = f(6, 8, 2, 32), i32(2, 3), i32(2), f(2, 2, 24)

    def refused(what, fn, *a, **o):
        with pytest.raises(AotHipError, match=what):
            fn(*a, **o)
    for fn, args in ((S.rope, (q, k, pos, freqs)), (S.masked_attention, (q, k, k)), (S.rope_append, (q[0], k[0], k[0], pos[0], freqs, pos[0], kp, kp)),
                     (S.paged_attention, (f(2, 4, 32), kp, kp, table, n)), (S.paged_evict, (kp, kp, table, n, w, i32(2, 1), 8))):
        refused('no CPU fallback', fn, *args)
    refused('pos', S.rope, q, k, pos.long(), freqs)
    refused('pos', S.rope, q, k, i32(1, 5), freqs)
    refused('freqs', S.rope, q, k, pos, freqs.float())
    refused('freqs', S.rope, q, k, pos, S.rope_freqs(34))
    refused('k must', S.rope, q, k.half(), pos, freqs)
    refused('float32 / float16', S.rope, q.double(), None, pos, freqs)
    refused('rot must', S.rope_freqs, 7)
    refused('stretch', S.rope_freqs, 8, stretch=0.5)
    refused('slots', S.rope_append, q[0], k[0], k[0], pos[0], freqs, pos[0].long(), kp, kp)
    refused('power of two', S.rope_append, q[0], k[0], k[0], pos[0], freqs, pos[0], f(6, 6, 2, 32), f(6, 6, 2, 32))
    refused('do not fit', S.rope_append, q[0], k[0], k[0], pos[0], freqs, pos[0], f(6, 8, 3, 32), f(6, 8, 3, 32))
    refused('do not fit', S.masked_attention, q, f(1, 4, 3, 32), f(1, 4, 3, 32))
    refused('head width', S.masked_attention, f(1, 4, 4, 136), f(1, 4, 2, 136), f(1, 4, 2, 136))
    refused('head width', S.masked_attention, f(1, 4, 4, 36).half(), f(1, 4, 2, 36).half(), f(1, 4, 2, 36).half())
    refused('go together', S.masked_attention, q, k, k, doc_q=pos)
    refused('doc_k', S.masked_attention, q, k, k, doc_q=pos, doc_k=i32(1, 3))
    refused('prefix', S.masked_attention, q, k, k, prefix=i32(2))
    refused('softcap', S.masked_attention, q, k, k, softcap=-1.0)
    refused('softcap', S.masked_attention, q, k, k, softcap=math.inf)
    refused('scale', S.masked_attention, q, k, k, scale=0.0)
    refused('scale', S.masked_attention, q, k, k, scale=-0.5)
    refused('scale', S.masked_attention, q, k, k, scale=math.nan)
    refused('softcap', S.paged_attention, f(2, 4, 32), kp, kp, table, n, softcap=math.nan)
    refused('beyond', S.paged_attention, f(1, 4, 32), f(1, 1 << 10, 2, 32), f(1, 1 << 10, 2, 32), i32(1, (1 << 20) + 1), i32(1))
    refused('slopes', S.masked_attention, q, k, k, slopes=f(3))
    refused('no gradient', S.masked_attention, q, k, k, slopes=f(4, requires_grad=True))
    refused('of one of', S.masked_attention, q, k, k.half())
    refused('weights', S.paged_attention, f(2, 4, 32), kp, kp, table, n, weights=f(2, 2, 23))
    refused('key_pos', S.paged_attention, f(2, 4, 32), kp, kp, table, n, key_pos=w)
    refused('table', S.paged_attention, f(2, 4, 32), kp, kp, table.long(), n)
    refused('lengths', S.paged_attention, f(2, 4, 32), kp, kp, table, i32(3))
    refused('query heads', S.paged_attention, f(2, 3, 32), kp, kp, table, n)
    refused('head width', S.paged_attention, f(2, 4, 264), f(6, 8, 2, 264), f(6, 8, 2, 264), table, n)
    refused('16-byte', S.paged_attention, f(2, 4, 32), f(6, 8, 2, 33)[..., :32], f(6, 8, 2, 33)[..., :32], table, n)
    refused('last dimension', S.paged_attention, f(2, 4, 32), f(6, 8, 32, 2).transpose(2, 3), f(6, 8, 32, 2).transpose(2, 3), table, n)
    refused('expanded', S.paged_attention, f(2, 4, 32), kp, kp, table, n, weights=f(1, 2, 24).expand(2, 2, 24))
    refused('expanded', S.rope_append, q[0], k[0], k[0], pos[0], freqs, pos[0], f(1, 8, 2, 32).expand(6, 8, 2, 32), kp)
    refused('expanded', S.paged_evict, kp, f(1, 8, 2, 32).expand(6, 8, 2, 32), table, n, w, i32(2, 1), 8)
    refused('serving call', S.paged_attention, f(2, 4, 32, requires_grad=True), kp, kp, table, n)
    refused('serving call', S.rope_append, q[0], f(4, 2, 32, requires_grad=True), k[0], pos[0], freqs, pos[0], kp, kp)
    refused('fit the budget', S.paged_evict, kp, kp, table, n, w, i32(2, 1), 8, sink=5, recent=4)
    refused('holds 8 entries', S.paged_evict, kp, kp, table, n, w, i32(2, 1), 9)
    refused('weights', S.paged_evict, kp, kp, table, n, f(2, 2, 23), i32(2, 1), 8)
    refused('key_pos', S.paged_evict, kp, kp, table, n, w, i32(2, 1), 8, key_pos=i32(2, 2, 23))


def test_stretched_frequencies():
    from networks.layers.sequence import rope_freqs
    plain, far = rope_freqs(64), rope_freqs(64, stretch=8.0)
    assert plain.dtype == torch.float64 and plain[0] == 1.0 and abs(float(plain[-1]) * 10000.0 ** (62 / 64) - 1) < 1e-12
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(far[turns >= 32], plain[turns >= 32]) and torch.allclose(far[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (far[mid] < plain[mid]).all() and (far[mid] > plain[mid] / 8).all()


def test_the_references_agree_with_torch():
    """The 64-bit references themselves, on the CPU, against torch's autograd and against each other."""
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(1, 9, n, 32, generator=g) for n in (4, 2, 2, 4))
    ids = torch.tensor([[0, 0, 1, 1, 1, 2, 2, -1, -1]], dtype=torch.int32)
    o, _, grads, _ = R.attention(q, k, v, do, causal=True, softcap=2.0, slopes=torch.full((4,), 0.1), doc_q=ids, doc_k=ids)
    x = [t.double().requires_grad_() for t in (q, k, v)]
    Q, K, V = x[0].transpose(1, 2), x[1].transpose(1, 2).repeat_interleave(2, 1), x[2].transpose(1, 2).repeat_interleave(2, 1)
    see, far = R.visible(1, 9, 9, True, ids, ids, None, 'cpu')
    s = 2.0 * torch.tanh(Q @ K.transpose(-1, -2) * 32 ** -0.5 / 2.0) - float(torch.tensor(0.1)) * far
    dead = ~see.any(-1)
    y = torch.softmax(s.masked_fill(~(see | dead[..., None])[:, None], float('-inf')), -1) @ V
    y = torch.where(dead[:, None, :, None], 0.0, y).transpose(1, 2)
    assert torch.allclose(y, o, atol=1e-13)
    for a, b in zip(torch.autograd.grad(y, x, do.double()), grads):
        assert torch.allclose(a, b, atol=1e-12)
    table, n = torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.tensor([9], dtype=torch.int32)
    kp, vp = torch.zeros(3, 4, 2, 32), torch.zeros(3, 4, 2, 32)
    for t in range(9):
        kp[table[0, t // 4], t % 4], vp[table[0, t // 4], t % 4] = k[0, t], v[0, t]
    a = R.paged(q[:, 8], kp, vp, table, n)[0]
    assert torch.allclose(a, R.attention(q, k, v, causal=True)[0][:, 8], atol=1e-13)
    assert R.evict(torch.tensor([[[1., 5., 5., 0., 7., float('nan')]]]), torch.tensor([6]), 4, 1, 1, 6) == [[0, 1, 4, 5]]


def test_cache_slots_of_padded_and_foreign_tokens():
    from networks.layers import sequence as S
    table = torch.tensor([[3, 0, 5], [1, -1, 1 << 28]], dtype=torch.int32)
    seq = torch.tensor([0, 0, 1, 0, -1, 2, 0, 1, 1])
    pos = torch.tensor([0, 47, 5, -1, 4, 4, 48, 17, 33], dtype=torch.int32)
    got = S.cache_slots(table, seq, pos, 16)
    assert got.dtype == torch.int32 and got.tolist() == [48, 95, 21, -1, -1, -1, -1, -1, -1]
    assert S.cache_slots(table[:, :0], seq, pos, 16).tolist() == [-1] * 9


@pytest.mark.parametrize('scale', [0.0, -0.5, math.inf, math.nan])
def test_one_token_attention_refuses_a_scale_that_is_not_positive(scale):
    import aot_hip
    from networks.layers import sequence as S
    P, i32 = ctypes.c_void_p, lambda *s: torch.zeros(s, dtype=torch.int32)
    strides = (ctypes.c_long * 15)()
    assert aot_hip.load().aot_paged_attn(P(16), P(16), P(16), P(16), P(16), None, None, None, P(16), None, 0, 0, 1, 1, 1, 32, 16, 1, 4, scale, 0.0,
                                         strides, None) == -1
    pages = torch.zeros(6, 8, 2, 32)
    with pytest.raises(aot_hip.AotHipError, match='scale must be positive'):
        S.paged_attention(torch.zeros(2, 4, 32), pages, pages, i32(2, 3), i32(2), scale=scale)
