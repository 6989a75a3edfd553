"""Rotary positions, masked attention, paged attention and eviction (networks/layers/sequence.py) on the MI355X, against their
definitions in 64 bits (tests/sequence_refs.py, where the bounds are derived)."""
import pytest
import torch

import sequence_refs as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def seq():
    assert torch.cuda.is_available(), 'GPU tests need a ROCm device'
    import aot_hip
    aot_hip.load()
    from networks.layers import sequence
    return sequence


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * scale).to(dtype)


def ints(lo, hi, shape, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device='cuda', dtype=torch.int32)


def within(name, got, want, bound):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), '%s: %d of %d values out, worst %.3g of a bound of %.3g' % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound.expand_as(off)[bad].min()))


# ---- rotary positions ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('S,H,K,D,rot,inter,far', [(1, 1, 1, 32, 32, False, 1), (5, 3, 1, 80, 20, True, 1000), (33, 4, 2, 128, 128, False, 1000000),
                                                   (7, 2, 2, 66, 34, False, 70000), (9, 5, 1, 256, 128, True, 2 ** 31 - 10), (3, 1, 1, 2, 2, True, 5),
                                                   (4100, 2, 1, 64, 64, False, 100)])
def test_rope_and_gradient(seq, dtype, S, H, K, D, rot, inter, far):
    dt, B = DT[dtype], 2
    q, k = rand((B, S, H, D), dt, 1).requires_grad_(), rand((B, S, K, D), dt, 2).requires_grad_()
    pos = ints(0, far, (B, S), 3)
    freqs = seq.rope_freqs(rot, stretch=4.0, device='cuda')
    yq, yk = seq.rope(q, k, pos, freqs, interleaved=inter, mscale=1.25)
    gq, gk = rand(q.shape, dt, 4), rand(k.shape, dt, 5)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    for name, x, y, sign in (('q', q, yq, 1), ('k', k, yk, 1), ('dq', gq, dq, -1), ('dk', gk, dk, -1)):
        want = R.turn(x.detach().double(), pos, freqs, inter, 1.25, sign)
        # the angle in 32-bit half turns in [-1, 1] (2^-25 of a half turn: pi 2^-25), its sine and cosine to a few steps, two products
        size = 1.25 * 1.5 * x.detach().double().abs().amax(-1, keepdim=True)
        tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
        within(name, y.detach(), want, R.half_step(dt) * want.abs() + 16 * R.E32 * size + tiny)
        if rot < D:
            assert torch.equal(y[..., rot:], x[..., rot:])


def test_rope_strides_one_tensor_and_shared_positions(seq):
    base = rand((2, 4, 9, 3 * 64), torch.bfloat16, 1)                    # [B, H, S, qkv]: q and k are slices
    q, k = base[..., :64].transpose(1, 2), base[..., 64:128].transpose(1, 2)
    pos = torch.arange(9, dtype=torch.int32, device='cuda')
    freqs = seq.rope_freqs(64, device='cuda')
    a, b = seq.rope(q, k, pos, freqs)
    c, d = seq.rope(q.contiguous(), k.contiguous(), pos.expand(2, 9).contiguous(), freqs)
    assert torch.equal(a, c) and torch.equal(b, d) and torch.equal(seq.rope(q, None, pos, freqs), a)
    off = torch.empty(2 * 9 * 4 * 64 + 1, dtype=torch.bfloat16, device='cuda')[1:].view(2, 9, 4, 64).copy_(q)      # misaligned rows
    for inter in (False, True):
        assert torch.equal(seq.rope(off, None, pos, freqs, interleaved=inter), seq.rope(q.contiguous(), None, pos, freqs, interleaved=inter))
    x = q.detach().requires_grad_()
    y = seq.rope(x, k, pos, freqs)[0]
    g, = torch.autograd.grad(y.float().sum(), x)                         # an expanded gradient
    within('sum gradient', g, R.turn(torch.ones(2, 9, 4, 64, dtype=torch.float64, device='cuda'), pos.expand(2, 9), freqs, sign=-1),
           torch.full((), 2 * R.half_step(torch.bfloat16), device='cuda'))
    e = seq.rope(q[:, :0], k[:, :0], pos[:0], freqs)
    assert e[0].shape == (2, 0, 4, 64)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('layout', ['place_head', 'head_place'])
def test_rope_append(seq, dtype, layout):
    dt, N, H, K, D, page, P = DT[dtype], 37, 6, 2, 48, 8, 12
    q, k, v = rand((N, H, D), dt, 1), rand((N, K, D), dt, 2), rand((N, K, D), dt, 3)
    pools = [rand((P, page, K, D) if layout == 'place_head' else (P, K, page, D), dt, 4 + i) for i in range(2)]
    kp, vp = pools if layout == 'place_head' else [x.transpose(1, 2) for x in pools]
    pos = ints(0, 200000, (N,), 5)
    slots = torch.randperm(P * page, device='cuda', generator=torch.Generator(device='cuda').manual_seed(6))[:N].to(torch.int32)
    slots[3] = -1
    slots[4] = P * page                                                   # outside the pool: nothing is written
    slots[5] = 2 ** 31 - 1
    freqs = seq.rope_freqs(32, device='cuda')
    for inter in (False, True):
        k0, v0 = kp.clone(), vp.clone()
        y = seq.rope_append(q, k, v, pos, freqs, slots, kp, vp, interleaved=inter)
        rq, rk = seq.rope(q[None], k[None], pos[None], freqs, interleaved=inter)
        ok = (slots >= 0) & (slots < P * page)
        at = slots[ok].long()
        k0[at // page, at % page], v0[at // page, at % page] = rk[0][ok], v[ok]
        assert torch.equal(y, rq[0]) and torch.equal(kp, k0) and torch.equal(vp, v0)
    assert seq.rope_append(None, k, v, pos, freqs, slots, kp, vp) is None
    table = torch.randperm(P, device='cuda').to(torch.int32).view(2, 6)
    s = seq.cache_slots(table, torch.tensor([0, 1, 1], device='cuda'), torch.tensor([0, 9, 47], device='cuda'), page)
    assert s.tolist() == [int(table[0, 0]) * 8, int(table[1, 1]) * 8 + 1, int(table[1, 5]) * 8 + 7] and s.dtype == torch.int32


# ---- masked attention ------------------------------------------------------------------------------------------------------------
def docs_of(B, S, n, seed, pad=0):
    ids = torch.sort(ints(0, n, (B, S), seed), dim=1).values.to(torch.int32)
    if pad:
        ids[:, S - pad:] = -1
    return ids


SHAPES = {            # B, Sq, Sk, H, K, D, options
    'one': (1, 1, 1, 1, 1, 32, {}),
    'one query': (2, 1, 300, 4, 1, 64, dict(causal=True)),
    'odd': (2, 77, 130, 6, 2, 40, dict(causal=True)),
    'plain': (1, 200, 333, 3, 3, 128, {}),
    'queries before the keys': (2, 190, 70, 2, 1, 64, dict(causal=True)),
    'capped': (1, 129, 129, 4, 4, 96, dict(causal=True, softcap=3.0)),
    'slopes': (1, 130, 260, 4, 2, 80, dict(slopes=True)),
    'documents': (2, 333, 333, 2, 2, 64, dict(causal=True, docs=5, pad=11)),
    'documents, no order': (2, 150, 150, 2, 1, 32, dict(docs=-4)),
    'prefix': (3, 140, 200, 2, 2, 64, dict(causal=True, prefix=True)),
    'everything': (2, 257, 257, 4, 2, 128, dict(causal=True, softcap=5.0, slopes=True, docs=3, pad=7, prefix=True)),
    'long row': (1, 3, 5001, 2, 1, 64, dict(causal=True)),
    'many queries': (1, 2000, 65, 2, 1, 32, dict(softcap=2.0)),
    'all padding': (1, 70, 70, 1, 1, 32, dict(docs=1, pad=70)),
}


def build(shape, dt, seed=0):
    B, Sq, Sk, H, K, D, o = SHAPES[shape]
    o = dict(o)
    q, k, v, do = rand((B, Sq, H, D), dt, seed + 1, 1.5), rand((B, Sk, K, D), dt, seed + 2), rand((B, Sk, K, D), dt, seed + 3), rand((B, Sq, H, D), dt, seed + 4)
    if o.pop('slopes', False):
        o['slopes'] = torch.rand(H, device='cuda', generator=torch.Generator(device='cuda').manual_seed(9)) * 0.1
    n, pad = o.pop('docs', 0), o.pop('pad', 0)
    if n:
        ids = docs_of(B, Sk, n, 11, pad) if n > 0 else ints(-1, -n, (B, Sk), 11)
        o['doc_q'] = o['doc_k'] = ids
    if o.pop('prefix', False):
        o['prefix'] = torch.tensor([50, 0, Sk + 5][:B], dtype=torch.int32, device='cuda')
    return q, k, v, do, o


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', SHAPES)
def test_masked_attention_and_gradients(seq, dtype, shape):
    q, k, v, do, o = build(shape, DT[dtype])
    lead = [x.requires_grad_() for x in (q, k, v)]
    out = seq.masked_attention(q, k, v, **o)
    grads = torch.autograd.grad(out, lead, do)
    again = torch.autograd.grad(seq.masked_attention(q, k, v, **o), lead, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), 'not repeatable'
    with torch.no_grad():
        want, bound, wg, bg = R.attention(q, k, v, do, **o)
    within('out', out.detach(), want, bound)
    for name, g, w, b in zip(('dq', 'dk', 'dv'), grads, wg, bg):
        within(name, g, w, b)


def test_prefix_outside_the_keys(seq):
    q, k, v = (rand((3, 40, 2, 64), torch.float32, i) for i in range(3))
    pre = torch.tensor([-2 ** 31, -1, 2 ** 31 - 1], dtype=torch.int32, device='cuda')
    out = seq.masked_attention(q, k, v, causal=True, prefix=pre)
    assert torch.equal(out[:2], seq.masked_attention(q[:2], k[:2], v[:2], causal=True))
    want, bound = R.attention(q[2:], k[2:], v[2:])
    within('all seen', out[2:], want, bound)


def test_calls_on_a_named_stream(seq):
    """stream=: the launch, its copies of odd inputs and its scratch belong to that stream."""
    import aot_hip
    x = rand((1, 700, 2, 3 * 64 + 1), torch.float16, 1)
    q, k, v = x[..., :64], x[..., 64:128], x[..., 128:192]                  # rows off 16 bytes: dense copies are made
    kp, vp, table, _ = cache(2, 4000, 16, 2, 64, torch.float16, 3)
    n = torch.tensor([4000, 77], dtype=torch.int32, device='cuda')
    want = aot_hip.attn_masked(q, k, v, causal=True)[0]
    wp = aot_hip.paged_attn(q[0, :2], kp, vp, table, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        a = aot_hip.attn_masked(q, k, v, causal=True, stream=side.cuda_stream)[0]
        b = aot_hip.paged_attn(q[0, :2], kp, vp, table, n, stream=side.cuda_stream)
        torch.empty(1 << 22, device='cuda').fill_(float('nan'))             # the current stream reuses what it may
    side.synchronize()
    assert torch.equal(a, want) and torch.equal(b, wp)


def test_masked_attention_empty_sides(seq):
    q, k = rand((2, 5, 2, 64), torch.float16, 1).requires_grad_(), rand((2, 0, 1, 64), torch.float16, 2).requires_grad_()
    out = seq.masked_attention(q, k, k, causal=True)
    dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
    assert not out.any() and not dq.any() and dk.shape == k.shape
    k = rand((2, 5, 1, 64), torch.float16, 3).requires_grad_()
    out = seq.masked_attention(q[:, :0], k, k)
    dk, = torch.autograd.grad(out, k, torch.ones_like(out))
    assert out.shape == (2, 0, 2, 64) and not dk.any()
    assert seq.masked_attention(q[:0], k[:0], k[:0]).shape == (0, 5, 2, 64)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('fill', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('more', [{}, dict(softcap=6.0), dict(softcap=6.0, slopes=True)])
def test_masked_places_may_hold_anything(seq, dtype, fill, more):
    """Results are those of the same call with zeros in the masked places, bit for bit."""
    dt = DT[dtype]
    S = 200
    ids = docs_of(1, S, 3, 5, 20)
    dead = ids[0] < 0
    if 'slopes' in more:
        more = dict(more, slopes=torch.tensor([0.02, 0.1], device='cuda'))
    late = torch.arange(S, device='cuda') >= 150                           # keys no query of a shorter query block sees

    def run(x):
        q, k, v, do = (rand((1, S, 2, 64), dt, 20 + i) for i in range(4))
        for t in (q, k, v, do):
            t[:, dead] = x
        lead = [t.requires_grad_() for t in (q, k, v)]
        a = seq.masked_attention(q, k, v, causal=True, doc_q=ids, doc_k=ids, **more)
        ga = torch.autograd.grad(a, lead, do)
        k2, v2 = rand((1, S, 2, 64), dt, 31), rand((1, S, 2, 64), dt, 32)
        k2[:, late], v2[:, late] = x, x
        q2, do2 = rand((1, S, 2, 64), dt, 33), rand((1, S, 2, 64), dt, 34)
        q2[:, late], do2[:, late] = x, x                                   # causal: rows before 150 see no late key; the late rows' results go
        lead2 = [t.requires_grad_() for t in (q2, k2, v2)]
        c = seq.masked_attention(q2, k2, v2, causal=True, **more)
        return [a] + list(ga), c[:, :150], torch.autograd.grad(c, lead2, do2)[0][:, :150]

    (a, c, dq), (a0, c0, dq0) = run(fill), run(0.0)
    for x, y in zip(a, a0):
        assert torch.isfinite(x).all() and torch.equal(x, y)
    assert torch.isfinite(c).all() and torch.equal(c, c0) and torch.equal(dq, dq0)


def test_seen_nan_reaches_the_result(seq):
    q, k, v = (rand((1, 100, 1, 64), torch.bfloat16, i) for i in range(3))
    v[0, 90, 0, 5] = float('nan')
    out = seq.masked_attention(q, k, v, causal=True)
    want = torch.zeros(100, 64, dtype=torch.bool, device='cuda')
    want[90:, 5] = True
    assert torch.equal(torch.isnan(out[0, :, 0]), want)


def test_masked_attention_strides_and_far_offsets(seq):
    dt = torch.bfloat16
    B, S, H, K, D = 2, 130, 4, 2, 64
    qkv = rand((B, S, (H + 2 * K) * D), dt, 1)
    q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([H * D, K * D, K * D], -1))          # slices of one projection
    do = rand((B, H, S, D), dt, 2).transpose(1, 2)

    def run(q, k, v, do):
        lead = [x.detach().requires_grad_() for x in (q, k, v)]
        out = seq.masked_attention(*lead, causal=True)
        return [out.detach()] + list(torch.autograd.grad(out, lead, do))
    want = run(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous())
    for a, b in zip(run(q, k, v, do), want):
        assert torch.equal(a, b)
    head_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    for a, b in zip(run(*head_first, do), want):
        assert torch.equal(a, b)
    odd = [torch.empty(x.numel() + 3, dtype=dt, device='cuda')[3:].view(x.shape).copy_(x) for x in (q, k, v)]    # rows off 16 bytes
    for a, b in zip(run(*odd, do), want):
        assert torch.equal(a, b)
    big = torch.empty(1 << 32, dtype=dt, device='cuda')                    # row strides past 2^31 elements in all
    far = torch.as_strided(big, (1, 300, 1, D), (0, 1 << 23, D, 1))
    kk, vv, qq = rand((1, 300, 1, D), dt, 5), rand((1, 300, 1, D), dt, 6), rand((1, 300, 1, D), dt, 7)
    a = run(qq, far.copy_(kk), vv, qq)
    b = run(qq, kk, vv, qq)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    big.zero_()
    a = run(qq, kk, far.copy_(vv), qq)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_masked_attention_against_differences(seq):
    """Directional derivatives of the definition (64 bits, central differences) against the kernel's gradients.  Truncation h^2 / 6 of a
    third derivative of order 1e2 at h = 1e-4: below 1e-6; the kernel's own error is under the bound of sequence_refs."""
    q, k, v, do, o = build('everything', torch.float32)
    lead = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(seq.masked_attention(q, k, v, **o), lead, do)
    with torch.no_grad():
        bounds = R.attention(q, k, v, do, **o)[3]
        for n in range(3):
            d = rand(lead[n].shape, torch.float64, 40 + n)

            def f(h):
                x = [t.double() for t in lead]
                x[n] = x[n] + h * d
                return float((R.attention(*x, **o)[0] * do.double()).sum())
            want = (f(1e-4) - f(-1e-4)) / 2e-4
            got = float((grads[n].double() * d).sum())
            assert abs(got - want) <= float((bounds[n] * d.abs()).sum()) + 1e-5 * max(1.0, abs(want)), (n, got, want)


# ---- paged attention ---------------------------------------------------------------------------------------------------------------
def cache(B, cap, page, K, D, dt, seed, spare=3, layout='place_head'):
    mp = -(-cap // page)
    P = B * mp + spare
    shape = (P, page, K, D) if layout == 'place_head' else (P, K, page, D)
    kp, vp = rand(shape, dt, seed), rand(shape, dt, seed + 1)
    if layout != 'place_head':
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    ids = torch.randperm(P, device='cuda', generator=torch.Generator(device='cuda').manual_seed(seed + 2)).to(torch.int32)
    return kp, vp, ids[:B * mp].view(B, mp).contiguous(), ids[B * mp:]


PAGED = {             # lengths, page, H, K, D, options
    'one entry': ([1], 16, 1, 1, 32, {}),
    'nothing': ([0, 5, 0], 4, 2, 1, 64, dict(weights=True)),
    'odd': ([1, 31, 32, 33, 127, 128, 129, 300], 16, 6, 2, 80, dict(weights=True)),
    'one place a page': ([77, 40], 1, 4, 4, 64, {}),
    'large page': ([700, 3], 512, 8, 1, 128, dict(softcap=4.0)),
    'many heads': ([260, 100], 32, 40, 2, 96, dict(weights=True, slopes=True)),
    'wide': ([513, 64], 64, 4, 2, 256, dict(slopes=True, softcap=10.0)),
    'wide and odd': ([200], 8, 3, 1, 136, {}),
    'long': ([70000, 1, 33000], 64, 8, 2, 64, dict(weights=True)),
    'positions': ([150, 90], 16, 4, 2, 64, dict(slopes=True, key_pos=True, weights=True)),
}


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('layout', ['place_head', 'head_place'])
@pytest.mark.parametrize('case', PAGED)
def test_paged_attention(seq, dtype, layout, case):
    dt = DT[dtype]
    lens, page, H, K, D, o = PAGED[case]
    if dt == torch.float32 and D == 136:
        D = 132                                                             # whole 16-byte pieces, not whole lanes' shares
    o = dict(o)
    B, cap = len(lens), max(max(lens), 1)
    kp, vp, table, _ = cache(B, cap, page, K, D, dt, 1, layout=layout)
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    S = table.shape[1] * page
    for b, n in enumerate(lens):                                            # whatever lies behind the length is not read
        t = torch.arange(n, S, device='cuda')
        kp[table[b].long()[t // page], t % page], vp[table[b].long()[t // page], t % page] = float('nan'), float('inf')
    q = rand((B, H, D), dt, 7, 1.5)
    if o.pop('slopes', False):
        o['slopes'] = torch.rand(H, device='cuda', generator=torch.Generator(device='cuda').manual_seed(8)) * 0.05
    if o.pop('key_pos', False):
        o['key_pos'] = torch.sort(ints(0, 5 * S, (B, K, S + 3), 9), -1).values.to(torch.int32)
    w0 = torch.rand(B, K, S + 1, device='cuda') if o.pop('weights', False) else None
    w = None if w0 is None else w0.clone()
    out = seq.paged_attention(q, kp, vp, table, lengths, weights=w, **o)
    want, bound, ww, bw = R.paged(q, kp, vp, table, lengths, **o)
    within('out', out, want, bound)
    for b, n in enumerate(lens):
        assert n or not out[b].any()
    if w is not None:
        within('weights', w[..., :S], w0[..., :S].double() + ww, bw + 2 * R.E32 * (w0[..., :S].double() + ww))
        assert torch.equal(w[..., S], w0[..., S])
        for b, n in enumerate(lens):
            assert torch.equal(w[b, :, n:], w0[b, :, n:]), 'entries past the length moved'
    out2 = torch.empty(B, 2 * H, D, dtype=dt, device='cuda')[:, ::2]
    assert seq.paged_attention(q, kp, vp, table, lengths, out=out2, **o) is out2 and (w is not None or torch.equal(out2, out))


def test_paged_attention_bad_pages_lengths_and_far_pools(seq):
    dt = torch.bfloat16
    kp, vp, table, _ = cache(2, 200, 16, 2, 64, dt, 1)
    q = rand((2, 4, 64), dt, 2)
    bad = table.clone()
    bad[0, 3], bad[0, 5], bad[1, 0] = -7, kp.shape[0], 2 ** 31 - 1
    lengths = torch.tensor([200, 190], dtype=torch.int32, device='cuda')
    w = torch.zeros(2, 2, table.shape[1] * 16, device='cuda')
    out = seq.paged_attention(q, kp, vp, bad, lengths, weights=w)
    want, bound, ww, bw = R.paged(q, kp, vp, bad, lengths)
    within('out', out, want, bound)
    within('weights', w, ww, bw + 1e-7 * ww)
    more = torch.tensor([10 ** 6, -5], dtype=torch.int32, device='cuda')      # past the table: all it holds; negative: nothing
    out = seq.paged_attention(q, kp, vp, table, more)
    full = seq.paged_attention(q, kp, vp, table, torch.full((2,), table.shape[1] * 16, dtype=torch.int32, device='cuda'))
    assert torch.equal(out[0], full[0]) and not out[1].any()
    assert not seq.paged_attention(q, kp[:0], vp[:0], table, lengths).any()      # an empty pool
    assert seq.paged_attention(q[:0], kp, vp, table[:0], lengths[:0]).shape == (0, 4, 64)
    pages = (1 << 31) // (64 * 2 * 64) + 40                                   # offsets past 2^31 elements
    big = [torch.empty(pages, 64, 2, 64, dtype=dt, device='cuda') for _ in range(2)]
    far = torch.tensor([[pages - 1, 0, pages - 7], [pages - 3, 5, 6]], dtype=torch.int32, device='cuda')
    near = torch.arange(6, dtype=torch.int32, device='cuda').view(2, 3)
    small = [rand((6, 64, 2, 64), dt, 3 + i) for i in range(2)]
    for b, s in zip(big, small):
        b[far.view(-1).long()] = s
    n = torch.tensor([190, 150], dtype=torch.int32, device='cuda')
    assert torch.equal(seq.paged_attention(q, *big, far, n), seq.paged_attention(q, *small, near, n))


# ---- eviction -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('lens,page,K,D,budget,sink,recent,kind', [
    ([40], 8, 1, 32, 10, 2, 3, 'random'), ([100, 10, 0, 33], 16, 3, 40, 33, 0, 0, 'ties'), ([300, 299], 4, 2, 64, 64, 64, 0, 'random'),
    ([500], 32, 2, 128, 100, 0, 100, 'same'), ([64, 20], 64, 2, 32, 20, 5, 5, 'nan'), ([5000, 1025], 64, 1, 36, 700, 4, 128, 'ties'),
    ([9], 1, 1, 32, 1, 0, 0, 'random'), ([777], 16, 2, 64, 776, 1, 1, 'zeros and signs')])
def test_paged_evict(seq, dtype, lens, page, K, D, budget, sink, recent, kind):
    dt = DT[dtype]
    B = len(lens)
    kp, vp, table, _ = cache(B, max(lens), page, K, D, dt, 1)
    more = -(-budget // page)
    kp, vp = (torch.cat([x, rand((B * more, page, K, D), dt, 5)]) for x in (kp, vp))
    new_table = (torch.arange(B * more, device='cuda') + kp.shape[0] - B * more).to(torch.int32).view(B, more)
    S = max(table.shape[1] * page, budget)
    w = torch.rand(B, K, S, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3))
    if kind == 'ties':
        w = (w * 4).floor()
    elif kind == 'same':
        w.fill_(0.5)
    elif kind == 'nan':
        w[..., ::3] = float('nan')
        w[..., 1::5] = float('inf')
    elif kind == 'zeros and signs':
        w = torch.where(w < 0.3, -w, torch.where(w < 0.6, torch.where(w < 0.45, 0.0, -0.0), w))
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    pos = torch.arange(S, dtype=torch.int32, device='cuda').expand(B, K, S) * 3 + 1
    k0, v0 = kp.clone(), vp.clone()
    kept, n, nw, np_ = seq.paged_evict(kp, vp, table, lengths, w, new_table, budget, sink, recent, key_pos=pos)
    rows = R.evict(w, lengths, budget, sink, recent, table.shape[1] * page)
    assert n.tolist() == [min(x, budget) for x in lens]
    j = torch.arange(S, device='cuda')
    for b in range(B):
        for h in range(K):
            want = torch.tensor(rows[b * K + h], dtype=torch.long, device='cuda')
            m = len(want)
            assert kept[b, h].tolist() == want.tolist() + [-1] * (budget - m)
            assert torch.equal(nw[b, h, :m].view(torch.int32), w[b, h, want].view(torch.int32)) and not nw[b, h, m:].any()
            assert torch.equal(np_[b, h, :m], pos[b, h, want]) and not np_[b, h, m:].any()
            src, at = table[b].long()[want // page], new_table[b].long()[j[:m] // page]
            for x, x0 in ((kp, k0), (vp, v0)):
                assert torch.equal(x[at, j[:m] % page, h], x0[src, want % page, h])
                x0[at, j[:m] % page, h] = x0[src, want % page, h]
    assert torch.equal(kp, k0) and torch.equal(vp, v0), 'something else was written'
    assert seq.paged_evict(kp, vp, table, lengths, w, new_table, budget, sink, recent)[3] is None
    k1 = kp.clone()
    off = torch.full_like(new_table, -1)                                       # nothing to move, the choice is reported
    off[0, 0] = kp.shape[0]
    assert torch.equal(seq.paged_evict(kp, vp, table, lengths, w, off, budget, sink, recent)[0], kept) and torch.equal(kp, k1)


# ---- together, streams, graphs --------------------------------------------------------------------------------------------------------
def serve(seq, dt, steps, graph_of=None):
    """Prompt, steps of one token with collected weights, an eviction half way, further steps: what a decoder does."""
    B, H, K, D, page, budget = 2, 4, 2, 64, 16, 48
    freqs = seq.rope_freqs(D, stretch=2.0, device='cuda')
    P = 24
    kp, vp = torch.zeros(P, page, K, D, dtype=dt, device='cuda'), torch.zeros(P, page, K, D, dtype=dt, device='cuda')
    table = torch.arange(16, dtype=torch.int32, device='cuda').view(B, 8)
    lens = [70, 41]
    w = torch.zeros(B, K, 128, device='cuda')
    kpos = torch.zeros(B, K, 128, dtype=torch.int32, device='cuda')
    row = torch.tensor([0] * lens[0] + [1] * lens[1], device='cuda')
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    q, k, v = rand((sum(lens), H, D), dt, 1), rand((sum(lens), K, D), dt, 2), rand((sum(lens), K, D), dt, 3)
    rq = seq.rope_append(q, k, v, pos, freqs, seq.cache_slots(table, row, pos, page), kp, vp)
    rk = kp[table.long()[row, pos.long() // page], pos.long() % page]
    prompt = seq.masked_attention(rq[None], rk[None], v[None], causal=True, doc_q=row.to(torch.int32)[None], doc_k=row.to(torch.int32)[None], softcap=20.0)
    kpos[:] = torch.arange(128, dtype=torch.int32, device='cuda')
    length = torch.tensor(lens, dtype=torch.int32, device='cuda')
    true = length.clone()                                                     # positions go on counting after an eviction
    outs = [prompt]
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625], device='cuda')
    history = []
    for s in range(steps):
        if s == steps // 2:
            new = torch.arange(16, 24, dtype=torch.int32, device='cuda').view(B, 4)
            kept, length, w, kpos = seq.paged_evict(kp, vp, table, length, w, new, budget, sink=2, recent=16, key_pos=kpos)
            table = torch.cat([new, table[:, 4:]], 1)                          # the old rows' last pages go on
            outs += [kept, w.clone()]
        q, k, v = rand((B, H, D), dt, 100 + s), rand((B, K, D), dt, 200 + s), rand((B, K, D), dt, 300 + s)
        slots = seq.cache_slots(table, torch.arange(B, device='cuda'), length, page)
        rq = seq.rope_append(q, k, v, true, freqs, slots, kp, vp)
        kpos.scatter_(2, length.long()[:, None, None].expand(B, K, 1), true[:, None, None].expand(B, K, 1))
        length, true = length + 1, true + 1
        history.append((rq, kp.clone(), vp.clone(), table.clone(), length.clone(), kpos.clone(), w.clone()))
        outs.append(seq.paged_attention(rq, kp, vp, table, length, softcap=20.0, slopes=slopes, weights=w, key_pos=kpos))
        history[-1] += (outs[-1], w.clone(), slopes)
    return outs, history


@pytest.mark.parametrize('dtype', DT)
def test_serving_run(seq, dtype):
    with torch.no_grad():
        outs, history = serve(seq, DT[dtype], 8)
        for rq, kp, vp, table, length, kpos, w0, out, w1, slopes in history:
            want, bound, ww, bw = R.paged(rq, kp, vp, table, length, softcap=20.0, slopes=slopes, key_pos=kpos)
            within('step', out, want, bound)
            within('weights', w1, w0.double() + ww, bw + 2 * R.E32 * (w0.double() + ww))
        again, _ = serve(seq, DT[dtype], 8)
        assert all(torch.equal(a, b) for a, b in zip(outs, again))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other, _ = serve(seq, DT[dtype], 8)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, other))


def test_training_run_together(seq):
    """rope -> masked attention -> loss, gradients of the projections' outputs against the 64-bit composition."""
    dt, B, S, H, K, D = torch.float32, 2, 150, 4, 2, 64
    q, k, v = (rand((B, S, n, D), dt, i).requires_grad_() for i, n in enumerate((H, K, K)))
    pos = torch.arange(S, dtype=torch.int32, device='cuda') + 90000
    freqs = seq.rope_freqs(D, device='cuda')
    ids = docs_of(B, S, 4, 3, 9)
    do = rand((B, S, H, D), dt, 9)
    rq, rk = seq.rope(q, k, pos, freqs)
    out = seq.masked_attention(rq, rk, v, causal=True, softcap=8.0, doc_q=ids, doc_k=ids)
    got = torch.autograd.grad(out, (q, k, v), do)
    with torch.no_grad():
        p2 = pos.expand(B, S)
        eq, ek = R.turn(q.double(), p2, freqs), R.turn(k.double(), p2, freqs)
        want, bound, g, b = R.attention(eq.float(), ek.float(), v, do, causal=True, softcap=8.0, doc_q=ids, doc_k=ids)
        g[0], g[1] = R.turn(g[0], p2, freqs, sign=-1), R.turn(g[1], p2, freqs, sign=-1)
    # the turned inputs differ by 16 steps of 2^-24: against gradients of order 1 through scores of order 10, 1e-4 of the largest
    for name, x, y in zip(('out', 'dq', 'dk', 'dv'), (out,) + got, [want] + g):
        assert float((x.detach().double() - y).abs().max()) <= 1e-4 * float(y.abs().max()), name


def test_graphs_replay_with_their_own_workspaces(seq):
    """Two captured steps (their workspaces live in the graphs' pools) replayed in turn with eager work between: each replay equals the
    eager call on the data it finds."""
    dt = torch.bfloat16
    kp, vp, table, _ = cache(2, 3000, 64, 2, 128, dt, 1)
    lengths = torch.tensor([3000, 1234], dtype=torch.int32, device='cuda')
    S = table.shape[1] * 64
    q = [rand((2, 8, 128), dt, 5 + i) for i in range(2)]
    w = [torch.zeros(2, 2, S, device='cuda') for _ in range(2)]
    x = [rand((1, 300, 2, 64), dt, 20 + i).requires_grad_() for i in range(3)]
    do = rand((1, 300, 2, 64), dt, 24)

    def step(i):
        return seq.paged_attention(q[i], kp, vp, table, lengths, weights=w[i])

    def train():
        out = seq.masked_attention(*x, causal=True, softcap=5.0)
        return (out,) + torch.autograd.grad(out, x, do)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        step(0)
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    for f in (lambda: step(0), lambda: step(1), train):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for rep in range(3):
        for t in q:
            t.copy_(rand(t.shape, dt, 50 + rep))
        lengths.copy_(torch.tensor([3000 - 700 * rep, 1 + rep], dtype=torch.int32))
        for t in w:
            t.zero_()
        for t in x:
            t.data.copy_(rand(t.shape, dt, 60 + rep))
        graphs[0].replay()
        graphs[1].replay()
        graphs[2].replay()
        torch.cuda.synchronize()
        got = [outs[0].clone(), outs[1].clone(), w[0].clone(), w[1].clone()] + [t.detach().clone() for t in outs[2]]
        for t in w:
            t.zero_()
        want = [step(0), step(1), w[0].clone(), w[1].clone()] + [t.detach() for t in train()]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_dispatcher_ops_are_the_same_calls(seq):
    import aot_hip_ops                                                        # noqa: F401
    ops = torch.ops.aot_hip
    dt = torch.float16
    q, k, v = (rand((1, 70, 2, 64), dt, i) for i in range(3))
    pos = torch.arange(70, dtype=torch.int32, device='cuda')[None]
    freqs = seq.rope_freqs(64, device='cuda')
    with torch.no_grad():
        a, b = ops.rope(q, k, pos, freqs, False, 1.0, False)
        c, d = seq.rope(q, k, pos, freqs)
        assert torch.equal(a, c) and torch.equal(b, d)
        out, lse, res = ops.attn_masked(q, k, v, None, True, 5.0, None, None, None, None, True)
        assert torch.equal(out, seq.masked_attention(q, k, v, causal=True, softcap=5.0)) and lse.shape == (1, 2, 70)
        g = ops.attn_masked_bwd(q, q, k, v, out, lse, res, None, True, 5.0, None, None, None, None)
        assert [x.shape for x in g] == [q.shape, k.shape, v.shape]
        kp, vp, table, _ = cache(2, 40, 16, 2, 64, dt, 3)
        n = torch.tensor([40, 7], dtype=torch.int32, device='cuda')
        w = [torch.zeros(2, 2, 48, device='cuda') for _ in range(2)]
        o = ops.paged_attn(q[0, :2], kp, vp, table, n, None, 0.0, None, w[0], None)
        assert torch.equal(o, seq.paged_attention(q[0, :2], kp, vp, table, n, weights=w[1])) and torch.equal(w[0], w[1])
        slots = torch.tensor([1, 5], dtype=torch.int32, device='cuda')
        t = ops.rope_append(q[0, :2], k[0, :2], v[0, :2], pos[0, :2], freqs, slots, kp, vp, False, 1.0)
        assert torch.equal(t, c[0, :2])
        new = torch.tensor([[6], [7]], dtype=torch.int32, device='cuda')
        r = ops.paged_evict(kp, vp, table, n, w[0], new, 8, 1, 2, None)
        e = seq.paged_evict(kp, vp, table, n, w[0], new, 8, 1, 2)
        assert all(torch.equal(x, y) for x, y in zip(r[:3], e[:3]))
