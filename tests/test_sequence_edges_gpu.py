"""Edges of the token-sequence operators on the MI355X, against their definitions in 64 bits (tests/sequence_refs.py, sequence_edge_refs.py)."""
import pytest
import torch

import sequence_edge_refs as X
import sequence_refs as R
from test_sequence_gpu import DT, cache, docs_of, rand, seq, within         # noqa: F401  (seq: the fixture)

pytestmark = pytest.mark.gpu


def results(seq, q, k, v, do, **o):                                        # noqa: F811
    lead = [x.detach().requires_grad_() for x in (q, k, v)]
    out = seq.masked_attention(*lead, **o)
    return [out.detach()] + list(torch.autograd.grad(out, lead, do))


# ---- eviction: rows longer than the registers hold, read again in every pass ------------------------------------------------------
@pytest.mark.parametrize('lens,page,K,budget,sink,recent,kind', [
    ([16384, 16383, 16321], 64, 2, 4096, 4, 128, 'random'), ([16385, 900, 1, 0], 64, 2, 4097, 0, 0, 'ties'), ([16385], 1, 1, 16384, 3, 5, 'random'),
    ([70000, 33333, 700, 65536], 16, 2, 5000, 7, 1000, 'random'), ([70001, 1023], 16, 1, 1000, 0, 0, 'ties'), ([40000], 256, 1, 640, 64, 0, 'same'),
    ([50000, 20001], 64, 1, 8191, 1, 1, 'nan'), ([131072, 130000], 64, 1, 4096, 4, 1024, 'nan')])
def test_paged_evict_of_long_rows(seq, lens, page, K, budget, sink, recent, kind):      # noqa: F811
    B, D, dt = len(lens), 8, torch.float16
    kp, vp, table, _ = cache(B, max(lens), page, K, D, dt, 1)
    more = -(-budget // page)
    kp, vp = (torch.cat([x, rand((B * more, page, K, D), dt, 5)]) for x in (kp, vp))
    new = (torch.arange(B * more, device='cuda') + kp.shape[0] - B * more).to(torch.int32).view(B, more)
    S = table.shape[1] * page
    w = torch.rand(B, K, S, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3))
    if kind == 'ties':
        w = (w * 4).floor()
    elif kind == 'same':
        w.fill_(0.5)
    elif kind == 'nan':
        w[..., ::3] = float('nan')
        w[..., 1::500] = float('inf')
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    pos = torch.arange(S, dtype=torch.int32, device='cuda').expand(B, K, S) * 3 + 1
    k0, v0 = kp.clone(), vp.clone()
    kept, n, nw, npos = seq.paged_evict(kp, vp, table, lengths, w, new, budget, sink, recent, key_pos=pos)
    rows = R.evict(w.cpu(), lengths.cpu(), budget, sink, recent, S)
    assert n.tolist() == [min(x, budget) for x in lens]
    j = torch.arange(budget, device='cuda')
    for b in range(B):
        for h in range(K):
            want = torch.tensor(rows[b * K + h], dtype=torch.long, device='cuda')
            m = len(want)
            assert torch.equal(kept[b, h, :m].long(), want) and bool((kept[b, h, m:] == -1).all())
            assert torch.equal(nw[b, h, :m].view(torch.int32), w[b, h, want].view(torch.int32)) and not nw[b, h, m:].any()
            assert torch.equal(npos[b, h, :m], pos[b, h, want]) and not npos[b, h, m:].any()
            src, at = table[b].long()[want // page], new[b].long()[j[:m] // page]
            for x0 in (k0, v0):
                x0[at, j[:m] % page, h] = x0[src, want % page, h]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


# ---- the cap, large and small ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('softcap', [1e-3, 0.5, 4.0, 20.0, 50.0, 1e3, 1e6, 1e8, 3e38])
@pytest.mark.parametrize('D,H,K,causal', [(64, 4, 2, True), (128, 2, 2, False), (32, 2, 1, True)])
def test_cap_of_any_size(seq, softcap, D, H, K, causal):                   # noqa: F811
    """In 32 bits, errors relative to the capped score and not to the cap; a cap far past the scores is no cap."""
    q, k, v, do = rand((1, 150, H, D), torch.float32, 1, 2.0), rand((1, 170, K, D), torch.float32, 2), rand((1, 170, K, D), torch.float32, 3), rand((1, 150, H, D), torch.float32, 4)
    got = results(seq, q, k, v, do, causal=causal, softcap=softcap)
    for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(q, k, v, do, causal=causal, softcap=softcap)):
        within(name, g, want, bound)
    if softcap >= 1e6:                                                      # (1 - (s / cap)^2 / 3 rounds to one)
        for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(q, k, v, do, causal=causal)):
            within(name, g, want, 2 * bound)


@pytest.mark.parametrize('dtype', DT)
def test_gradients_of_scores_near_the_cap(seq, dtype):                      # noqa: F811
    """Every score three to eight times the cap: the cap's derivative is 1e-2 to 1e-6 and keeps its relative accuracy, on both sides of zero."""
    dt = DT[dtype]
    q, k, v, do = (rand((1, 70, 2, 64), dt, i) for i in range(4))
    side = torch.where(torch.arange(70, device='cuda') % 2 == 0, 1.0, -1.0)
    q, k = (0.02 * q.float() + 1.0).to(dt), ((0.02 * k.float() + 1.0) * side[None, :, None, None]).to(dt)      # scores near +-8
    for softcap in (1.0, 2.5):
        got = results(seq, q, k, v, do, softcap=softcap)
        for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(q, k, v, do, softcap=softcap)):
            within(name, g, want, bound)


@pytest.mark.parametrize('softcap', [1e-3, 20.0, 1e3, 1e6, 3e38])
@pytest.mark.parametrize('D', [32, 128, 256])
def test_cap_of_any_size_over_pages(seq, softcap, D):                       # noqa: F811
    kp, vp, table, _ = cache(2, 700, 16, 2, D, torch.float32, 1)
    q, lengths = rand((2, 4, D), torch.float32, 7, 2.0), torch.tensor([700, 333], dtype=torch.int32, device='cuda')
    w = torch.zeros(2, 2, table.shape[1] * 16, device='cuda')
    out = seq.paged_attention(q, kp, vp, table, lengths, softcap=softcap, weights=w)
    for b, n in enumerate(lengths.tolist()):
        t = torch.arange(n, device='cuda')
        k, v = (x[table[b].long()[t // 16], t % 16][None] for x in (kp, vp))
        want, bound = X.attention(q[b][None, None], k, v, torch.zeros_like(q[b])[None, None], softcap=softcap)[0]
        within('out', out[b][None, None], want, bound + 16 * R.E32 * want.abs())      # (the join over splits)
        unit = torch.eye(n, device='cuda')[None, :, None].expand(1, n, 2, n)             # values of unit vectors: the probabilities themselves
        p, bound = X.attention(q[b][None, None], k, unit, torch.zeros(1, 1, 4, n, device='cuda'), softcap=softcap)[0]
        within('weights', w[b, :, :n], p[0, 0].unflatten(0, (2, 2)).sum(1), (bound + 16 * R.E32 * p)[0, 0].unflatten(0, (2, 2)).sum(1))


# ---- infinities and NaN in places that are seen -------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('Sq,D', [(70, 64), (130, 128), (1, 32), (65, 32)])
def test_a_key_of_weight_zero_takes_no_gradient(seq, dtype, Sq, D):         # noqa: F811
    """A seen key whose infinite element makes every score -inf: weight zero, gradients zero, whether or not the queries fill their tiles."""
    dt, t = DT[dtype], 40
    q, k, v, do = rand((1, Sq, 2, D), dt, 1), rand((1, 100, 1, D), dt, 2), rand((1, 100, 1, D), dt, 3), rand((1, Sq, 2, D), dt, 4)
    q[..., 5] = -q[..., 5].abs() - 0.01
    k[0, t, 0, 5] = float('inf')
    rest = torch.arange(100, device='cuda') != t
    out, dq, dk, dv = results(seq, q, k, v, do)
    ref = X.attention(q, k[:, rest], v[:, rest], do)
    within('out', out, *ref[0])
    cols = torch.arange(D, device='cuda') != 5                                 # (dq's own column is 0 * inf)
    within('dq', dq[..., cols], *(x[..., cols] for x in ref[1]))
    for name, g, r in (('dk', dk, ref[2]), ('dv', dv, ref[3])):
        assert not g[:, t].any(), name
        within(name, g[:, rest], *r)


def same_kind(name, got, want, bound):
    """NaN and infinities at the same places, finite values within their bound."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), '%s: NaN at %d places for %d' % (name, int(torch.isnan(got).sum()), int(torch.isnan(want).sum()))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got.double()[inf], want[inf]), '%s: infinities' % name
    ok = torch.isfinite(want)
    within(name, got[ok], want[ok], bound[ok])


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('fill', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('which', ['q', 'k', 'v', 'do'])
@pytest.mark.parametrize('softcap', [0.0, 5.0])
@pytest.mark.parametrize('causal,D', [(True, 64), (True, 128), (False, 32)])
def test_seen_infinities_and_nan_in_the_gradients(seq, dtype, fill, which, softcap, causal, D):      # noqa: F811
    """One non-finite element that some queries see: the same results as the definition's, in a tile with a mask and in one without.  (Scores of
    order 1, so no probability that counts is too small for 32 bits.)"""
    dt = DT[dtype]
    for place in (3, 75, 139):                                             # whole tiles above it; inside a masked one; the last row of all
        x = dict(q=rand((1, 140, 2, D), dt, 1, 0.7), k=rand((1, 140, 1, D), dt, 2, 0.7), v=rand((1, 140, 1, D), dt, 3), do=rand((1, 140, 2, D), dt, 4))
        x[which][0, place, 0, 6] = fill
        got = results(seq, x['q'], x['k'], x['v'], x['do'], causal=causal, softcap=softcap)
        for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(x['q'], x['k'], x['v'], x['do'], causal=causal, softcap=softcap)):
            same_kind('%s, %s at %d' % (name, which, place), g, want, bound)


@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('which', ['q', 'k', 'v', 'do'])
def test_seen_infinities_where_the_sides_are_split(seq, dtype, which):      # noqa: F811
    """Few queries over many keys: several workgroups share a block's tiles, one of them meets the element."""
    dt = DT[dtype]
    for place in (5, 130):
        x = dict(q=rand((1, 140, 2, 32), dt, 1, 0.7), k=rand((1, 1100, 1, 32), dt, 2, 0.7), v=rand((1, 1100, 1, 32), dt, 3), do=rand((1, 140, 2, 32), dt, 4))
        at = place if which in ('q', 'do') else 960 + place
        x[which][0, at, 0, 6] = float('inf')
        got = results(seq, x['q'], x['k'], x['v'], x['do'], causal=True, softcap=5.0)
        for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(x['q'], x['k'], x['v'], x['do'], causal=True, softcap=5.0)):
            same_kind('%s, %s at %d' % (name, which, at), g, want, bound)


@pytest.mark.parametrize('dtype', DT)
def test_seen_infinities_within_documents(seq, dtype):                      # noqa: F811
    dt, D = DT[dtype], 64
    ids = docs_of(1, 200, 4, 5, 13)
    for which in range(4):
        x = [rand((1, 200, 2, D), dt, 1, 0.7), rand((1, 200, 2, D), dt, 2, 0.7), rand((1, 200, 2, D), dt, 3), rand((1, 200, 2, D), dt, 4)]
        x[which][0, 100, 1, 9] = float('inf')
        for t in x:
            t[0, 190] = float('nan')                                        # padding
        got = results(seq, *x, causal=True, softcap=4.0, doc_q=ids, doc_k=ids)
        for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(*x, causal=True, softcap=4.0, doc_q=ids, doc_k=ids)):
            same_kind('%s of %d' % (name, which), g, want, bound)


# ---- fp16: small gradients, small probabilities ---------------------------------------------------------------------------------------
def rounded_once(got, want, bound, name):
    """Elementwise within the bound, which an answer of zeros is not; and over all not twice as far off as the definition rounded once (the
    score gradient's or the probability's own rounding adds an independent error of the same relative size: 1.4)."""
    within(name, got, want, bound)
    assert float((want.abs() > bound).double().mean()) > 0.5, name + ': the bound is too wide to say anything'
    once = (want.half().double() - want).norm()
    assert float((got.double() - want).norm()) <= 2 * float(once), name


@pytest.mark.parametrize('size', [1.0, 1e-3, 1e-4])
@pytest.mark.parametrize('Sq,Sk,H,K,D,o', [(256, 4096, 2, 1, 64, {}), (300, 2500, 2, 2, 128, dict(causal=True)), (200, 3000, 2, 2, 32, dict(softcap=5.0)),
                                           (512, 6000, 4, 2, 64, dict(causal=True))])
def test_small_gradients_in_fp16(seq, size, Sq, Sk, H, K, D, o):            # noqa: F811
    dt = torch.float16
    q, k, v, do = rand((1, Sq, H, D), dt, 1), rand((1, Sk, K, D), dt, 2), rand((1, Sk, K, D), dt, 3), rand((1, Sq, H, D), dt, 4, size)
    got = results(seq, q, k, v, do, **o)
    ref = X.attention(q, k, v, do, **o)
    within('out', got[0], *ref[0])
    for name, g, (want, bound) in zip(('dq', 'dk', 'dv'), got[1:], ref[1:]):
        rounded_once(g, want, bound, name)


def test_gradients_of_rows_far_apart_in_fp16(seq):                          # noqa: F811
    """Documents whose gradients differ by 1e6, and rows of one document by 1e3: every row of dq and every document's dk keeps its digits."""
    dt, S = torch.float16, 700
    ids = docs_of(1, S, 3, 5)
    q, k, v = (rand((1, S, 2, 64), dt, i) for i in range(3))
    size = torch.where(ids[0] == 1, 1e-4, 100.0) * torch.where(torch.arange(S, device='cuda') % 3 == 0, 1.0, 1e-3 ** 0.5)
    do = (rand((1, S, 2, 64), torch.float32, 4) * size[None, :, None, None]).to(dt)
    got = results(seq, q, k, v, do, causal=True, doc_q=ids, doc_k=ids)
    for name, g, (want, bound) in zip(('out', 'dq', 'dk', 'dv'), got, X.attention(q, k, v, do, causal=True, doc_q=ids, doc_k=ids)):
        within(name, g, want, bound)
        for d in range(3):
            r = ids[0] == d
            assert float((g[0, r].double() - want[0, r]).norm()) <= 2 * float((want[0, r].half().double() - want[0, r]).norm()), (name, d)


def test_values_gradient_over_a_long_row_in_fp16(seq):                      # noqa: F811
    """Probabilities of 2^-17: normal numbers of their product, not subnormal ones of seven bits."""
    dt = torch.float16
    q, k, v, do = rand((1, 64, 1, 32), dt, 1, 0.5), rand((1, 1 << 17, 1, 32), dt, 2, 0.5), rand((1, 1 << 17, 1, 32), dt, 3), rand((1, 64, 1, 32), dt, 4, 100.0)
    got, ref = results(seq, q, k, v, do), X.attention(q, k, v, do)
    rounded_once(got[3], *ref[3], 'dv')


def spread(Sk, D, every):
    """Queries of 1 and keys whose scores are 25.5 ln 2 at every so-many-th place and 0 elsewhere; values there 0, elsewhere about 1000."""
    top = 25.5 * 0.6931471805599453 / D ** 0.5
    k = torch.zeros(1, Sk, 1, D, device='cuda')
    k[:, ::every] = top
    v = rand((1, Sk, 1, D), torch.float32, 3) * 100 + 1000
    v[:, ::every] = 0
    return torch.ones(1, 3, 1, D, device='cuda').half(), k.half(), v.half()


def test_many_small_probabilities_in_fp16(seq):                             # noqa: F811
    """A few keys take nearly all the weight; what the thousands of others share, 2^-25 of theirs each, is the whole result."""
    q, k, v = spread(8192, 64, 64)
    ref = X.attention(q, k, v, torch.zeros_like(q))[0]
    out = seq.masked_attention(q, k, v)
    within('out', out, *ref)
    assert float((ref[0].abs() > 4 * ref[1]).double().mean()) > 0.9
    q, k, v = spread(8192, 64, 32)
    ref = X.attention(q[:, :1], k, v, torch.zeros_like(q[:, :1]))[0]
    table = torch.arange(128, dtype=torch.int32, device='cuda').view(1, 128)
    w = torch.zeros(1, 1, 8192, device='cuda')
    n = torch.tensor([8192], dtype=torch.int32, device='cuda')
    for weights in (None, w):
        out = seq.paged_attention(q[0, :1], k.view(128, 64, 1, 64), v.view(128, 64, 1, 64), table, n, weights=weights)
        within('paged', out[None], *ref)
    want, bound = R.paged(q[0, :1], k.view(128, 64, 1, 64), v.view(128, 64, 1, 64), table, n)[2:]
    within('weights', w, want, bound)


# ---- rotary rows: one, two or four a workgroup -----------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('S,inter', [(4097, False), (16387, True), (16385, False)])
def test_rotary_rows_a_workgroup(seq, dtype, S, inter):                     # noqa: F811
    """Odd numbers of rows where a workgroup takes several: the same bits as the rows in short calls, appended too."""
    dt = DT[dtype]
    q, k = rand((S, 2, 32), dt, 1), rand((S, 1, 32), dt, 2)
    pos, freqs = torch.arange(S, dtype=torch.int32, device='cuda') * 7, seq.rope_freqs(20, device='cuda')
    a, b = seq.rope(q[None], k[None], pos, freqs, interleaved=inter)
    short = [seq.rope(q[None, i:i + 1000], k[None, i:i + 1000], pos[i:i + 1000], freqs, interleaved=inter) for i in range(0, S, 1000)]
    assert torch.equal(a, torch.cat([x for x, _ in short], 1)) and torch.equal(b, torch.cat([x for _, x in short], 1))
    pages = [torch.zeros(S // 16 + 1, 16, 1, 32, dtype=dt, device='cuda') for _ in range(2)]
    slots = torch.arange(S, dtype=torch.int32, device='cuda')
    t = seq.rope_append(q, k, k, pos, freqs, slots, *pages, interleaved=inter)
    assert torch.equal(t, a[0]) and torch.equal(pages[0].view(-1, 1, 32)[:S], b[0]) and torch.equal(pages[1].view(-1, 1, 32)[:S], k)
    assert not pages[0].view(-1, 1, 32)[S:].any()
