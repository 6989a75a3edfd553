"""Masked attention in 64 bits once more, for its edges: every sum runs over the seen pairs alone, infinities and NaN go through it as IEEE
arithmetic has them, and the bounds are relative to what they bound (tests/test_sequence_edges_gpu.py).

Steps counted: u = finfo.eps / 2 of the inputs' type for each rounding to it, 2^-24 for a 32-bit operation.
  score   a sum of D products, the scale and its powers of two: (D + 8) 2^-24 of the products' magnitudes; the cap, whatever its size, 16 2^-24 of
          the capped score; the bias 4 2^-24 of itself; the exponent 4 2^-24 of the score and (16 + Sk / 16) 2^-24 for exp2, rescales and sums.
  p       relative to itself, its own score's error and the normaliser's.  One rounding to the type, u p; in fp16 p is held 2^15 times as large,
          so that what falls below its smallest step is half of 2^-24 2^-15.
  ds      one rounding, u ds; in fp16 held so that a row's largest is in (2^14, 2^15]: below the smallest step 2^-25 / 2^14 of the largest is lost.
  cap'    4 E / (1 + E)^2, E = e^-2|y|: 16 2^-24 of itself and twice the error of y = s / cap; an E below the smallest normal number, 2^-126, may be
          taken for zero, which is 2^-124.
  result  one rounding: u of the value, and in fp16 half of its smallest step, 2^-25."""
import torch

from sequence_refs import E32, half_step, visible


def finite(x):
    return torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)


def pair_sum(a, b, see=None):
    """sum_j a[.., i, j] b[.., j, d] over the seen j: what lies at unseen pairs is never multiplied."""
    if bool(torch.isfinite(a).all()) and bool(torch.isfinite(b).all()):
        return (a if see is None else torch.where(see, a, 0.0)) @ b
    x = a.unsqueeze(-1) * b.unsqueeze(-3)
    return (x if see is None else torch.where(see.unsqueeze(-1), x, 0.0)).sum(-2)


def attention(q, k, v, do, scale=None, causal=False, softcap=0.0, slopes=None, doc_q=None, doc_k=None, prefix=None):
    """(out, bound), (dq, bound), (dk, bound), (dv, bound); q, do [B, Sq, H, D], k, v [B, Sk, Hk, D]."""
    u, half = half_step(q.dtype), q.dtype == torch.float16
    once = 2.0 ** -25 if half else 0.0
    B, Sq, H, D = q.shape
    Sk, K = k.shape[1:3]
    G = H // K
    scale = D ** -0.5 if scale is None else scale
    see, far = visible(B, Sq, Sk, causal, doc_q, doc_k, prefix, q.device)
    see = see[:, None].expand(B, H, Sq, Sk)
    Q, dO = (x.double().transpose(1, 2) for x in (q, do))
    Kx, V = (x.double().transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    T = lambda x: x.transpose(-1, -2)                                     # noqa: E731
    y = pair_sum(Q, T(Kx)) * scale
    mag = finite(Q).abs() @ T(finite(Kx).abs()) * scale
    es, s, slope = (D + 8) * E32 * mag, y, torch.ones_like(y)
    if softcap:
        th = torch.tanh(y / softcap)
        s = softcap * th
        e = torch.exp(-2 * (y / softcap).abs())
        slope = 4 * e / (1 + e) ** 2
        rel = 16 * E32 + 2 * es / softcap                                  # of the cap's derivative
        es = es * finite(slope) + 16 * E32 * finite(s).abs()
    else:
        rel = torch.zeros_like(es)
    if slopes is not None:
        b = slopes.double()[:, None, None] * far
        s = s - b
        es = es + 4 * E32 * b
    es = es + 4 * E32 * finite(s).abs() + (16 + Sk / 16) * E32
    s = torch.where(see, s, float('-inf'))
    m = s.amax(-1, keepdim=True)
    p = torch.where(see, torch.exp(s - torch.where(m == float('-inf'), 0.0, m)), 0.0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    P = finite(p)
    ep = es + (P * es).sum(-1, keepdim=True)
    o = pair_sum(p, V, see)
    aV, aK, aQ, aO = (finite(x).abs() for x in (V, Kx, Q, dO))
    bo = (P * (u + ep)) @ aV + u * finite(o).abs() + (2.0 ** -40 * (see.double() @ aV) if half else 0.0)
    dp = pair_sum(dO, T(V))
    delta = (dO * o).sum(-1, keepdim=True)
    ds = torch.where(see, p * (dp - delta) * slope, 0.0)
    adp = finite(dp).abs() + finite(delta).abs()
    edelta = (aO * (bo + once)).sum(-1, keepdim=True) + (D + 8) * E32 * (aO * finite(o).abs()).sum(-1, keepdim=True)
    c = finite(slope)
    eds = u * finite(ds).abs() + P * c * ((D + 8) * E32 * (aO @ T(aV)) + edelta) + P * adp * (c * (ep + rel) + (2.0 ** -124 if softcap else 0.0))
    fold = lambda x: x.unflatten(1, (K, G)).sum(2)                         # noqa: E731
    top = finite(ds).abs()
    lost = 2.0 ** -39 if half else 0.0
    eq = torch.where(see, eds + lost * top.amax(-1, keepdim=True), 0.0)
    ek = torch.where(see, eds + lost * top.amax(-2, keepdim=True).unflatten(1, (K, G)).amax(2, keepdim=True).expand(B, K, G, 1, Sk).flatten(1, 2), 0.0)
    ev = torch.where(see, P * (u + ep) + (2.0 ** -40 if half else 0.0), 0.0)
    sums = (64 + max(Sq, Sk) / 8) * E32                                     # the 32-bit sums over rows

    def result(x, bound, size):
        bound = bound + sums * size
        return x.transpose(1, 2), (bound + u * (finite(x).abs() + bound) + once).transpose(1, 2)
    return [(o.transpose(1, 2), (bo + once).transpose(1, 2)),
            result(pair_sum(ds, Kx, see) * scale, eq @ aK * scale, top @ aK * scale),
            result(fold(pair_sum(T(ds), Q, T(see))) * scale, fold(T(ek) @ aQ) * scale, fold(T(top) @ aQ) * scale),
            result(fold(pair_sum(T(p), dO, T(see))), fold(T(ev) @ aO), fold(T(P) @ aO))]
