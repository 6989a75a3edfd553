"""The token-sequence operators in 64 bits, with elementwise bounds on what a kernel's roundings may do (tests/test_sequence_*.py).

Bounds count steps: u = finfo.eps / 2 of the inputs' type for a value rounded to it once, 2^-24 for one 32-bit operation.  A score is a
sum of D products (D 2^-24 of the sum of their magnitudes), a cap and a scale on top, and its error moves the probability by that
much relative; exp2, the running rescales and the sum add a few 2^-24 for every tile of 64 keys."""
import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turn(x, pos, freqs, interleaved=False, mscale=1.0, sign=1):
    """x [..., S, H, D] float64, pos [..., S]."""
    n = 2 * freqs.numel()
    a = pos.double().unsqueeze(-1).unsqueeze(-1) * freqs * sign
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale
    y = x.clone()
    if interleaved:
        u, w = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = u * c - w * s, w * c + u * s
    else:
        u, w = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = u * c - w * s, w * c + u * s
    return y


def visible(B, Sq, Sk, causal, doc_q, doc_k, prefix, dev):
    i = torch.arange(Sq, device=dev)[:, None] + Sk - Sq
    t = torch.arange(Sk, device=dev)[None]
    see = torch.ones(B, Sq, Sk, dtype=torch.bool, device=dev)
    if causal:
        see = (t <= i).expand(B, Sq, Sk)
        if prefix is not None:
            see = see | (t[None] < prefix[:, None, None])
    if doc_q is not None:
        see = see & (doc_q[:, :, None] == doc_k[:, None, :]) & (doc_q[:, :, None] >= 0)
    return see, (i - t).abs().double()


def attention(q, k, v, do=None, scale=None, causal=False, softcap=0.0, slopes=None, doc_q=None, doc_k=None, prefix=None):
    """(out, out's bound, [dq, dk, dv], [their bounds]) in float64, out [B, Sq, H, D]."""
    u = half_step(q.dtype)
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 0.0            # half of fp16's smallest step
    B, Sq, H, D = q.shape
    Sk, K = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    see, far = visible(B, Sq, Sk, causal, doc_q, doc_k, prefix, q.device)
    see = see[:, None]
    clean = lambda x, ok: torch.where(ok[:, :, None, None], x.double(), 0.0)      # noqa: E731  rows nobody sees: whatever they hold
    Q = clean(q, see.any(-1)[:, 0]).transpose(1, 2)
    Kx = clean(k, see.any(-2)[:, 0]).transpose(1, 2).repeat_interleave(H // K, 1)
    V = clean(v, see.any(-2)[:, 0]).transpose(1, 2).repeat_interleave(H // K, 1)
    s = Q @ Kx.transpose(-1, -2) * scale
    mag = Q.abs() @ Kx.abs().transpose(-1, -2) * abs(scale)
    es = (D + 8) * E32 * mag
    th = torch.zeros_like(s)
    if softcap:
        th = torch.tanh(s / softcap)
        s = softcap * th
        es = es + 16 * E32 * softcap
    if slopes is not None:
        b = slopes.double()[:, None, None] * far
        s = s - b
        es = es + 4 * E32 * b
    es = es + 4 * E32 * s.abs() + (16 + Sk / 16) * E32
    s = torch.where(see, s, float('-inf'))
    m = s.amax(-1, keepdim=True) if Sk else s.new_zeros(B, H, Sq, 1)
    p = torch.exp(s - torch.where(m == float('-inf'), 0.0, m))
    p = torch.where(see, p, 0.0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    ep = es + (p * es).sum(-1, keepdim=True)                            # relative: its own score's and the normaliser's
    o = p @ V
    bo = (p * (u + ep)) @ V.abs() + u * o.abs() + tiny * (1 + V.abs().sum(-2, keepdim=True))
    back = lambda x: x.transpose(1, 2)                                  # noqa: E731
    if do is None:
        return back(o), back(bo)
    dO = clean(do, see.any(-1)[:, 0]).transpose(1, 2)
    dp = dO @ V.transpose(-1, -2)
    delta = (dO * o).sum(-1, keepdim=True)
    cap = 1 - th * th
    ds = p * (dp - delta) * cap
    edp = (D + 8) * E32 * (dO.abs() @ V.abs().transpose(-1, -2))
    edelta = (dO.abs() * (bo + u * o.abs())).sum(-1, keepdim=True) + (D + 8) * E32 * (dO * o).abs().sum(-1, keepdim=True)
    eds = u * ds.abs() + p * cap * (edp + edelta) + p * (dp.abs() + delta.abs()) * (ep * cap + (16 * E32 + 2 * es / softcap if softcap else 0.0)) + tiny
    eds = torch.where(see, eds, 0.0)
    dq, bq = ds @ Kx * scale, (eds @ Kx.abs() * abs(scale))
    dk, bk = ds.transpose(-1, -2) @ Q * scale, (eds.transpose(-1, -2) @ Q.abs()) * abs(scale)
    dv, bv = p.transpose(-1, -2) @ dO, (p * (u + ep) + tiny * see).transpose(-1, -2) @ dO.abs()
    fold = lambda x: x.unflatten(1, (K, H // K)).sum(2)                 # noqa: E731
    acc = (64 + Sq / 8) * E32                                           # the 32-bit sums over rows
    grads, bounds = [], []
    for g, b, shared, absum in ((dq, bq, False, ds.abs() @ Kx.abs() * abs(scale)), (dk, bk, True, ds.abs().transpose(-1, -2) @ Q.abs() * abs(scale)),
                                (dv, bv, True, p.transpose(-1, -2) @ dO.abs())):
        b = b + acc * absum
        if shared:
            g, b = fold(g), fold(b)
        grads.append(back(g))
        bounds.append(back(b + u * (g.abs() + b) + tiny))
    return back(o), back(bo), grads, bounds


def paged(q, k_pages, v_pages, table, lengths, scale=None, softcap=0.0, slopes=None, key_pos=None):
    """(out, bound, weights [B, K, cap] of this call, bound) in float64."""
    B, H, D = q.shape
    P, page, K, _ = k_pages.shape
    cap = table.shape[1] * page
    u = half_step(q.dtype)
    tiny = 2.0 ** -24 if q.dtype == torch.float16 else 0.0
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    w = torch.zeros(B, K, cap, dtype=torch.float64, device=q.device)
    bw = torch.zeros_like(w)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        if n == 0:
            continue
        t = torch.arange(n, device=q.device)
        pg = table[b].long()[t // page]
        ok = (pg >= 0) & (pg < P)
        pg = pg.clamp(0, max(P - 1, 0))
        for h in range(K):
            g = slice(h * (H // K), (h + 1) * (H // K))
            kk = torch.where(ok[:, None], k_pages[pg, t % page, h].double(), 0.0)
            vv = torch.where(ok[:, None], v_pages[pg, t % page, h].double(), 0.0)
            s = q[b, g].double() @ kk.T * scale
            es = (D + 8) * E32 * (q[b, g].double().abs() @ kk.abs().T) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                es = es + 16 * E32 * softcap
            if slopes is not None:
                at = key_pos[b, h, :n] if key_pos is not None else t
                far = (at[n - 1] - at).abs().double()
                s = s - slopes.double()[g, None] * far
                es = es + 4 * E32 * slopes.double()[g, None] * far
            es = es + 4 * E32 * s.abs() + (32 + n / 16) * E32
            s = torch.where(ok, s, float('-inf'))
            m = s.amax(-1, keepdim=True)
            p = torch.where(ok, torch.exp(s - torch.where(m == float('-inf'), 0.0, m)), 0.0)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            ep = es + (p * es).sum(-1, keepdim=True)
            out[b, g] = p @ vv
            bound[b, g] = (p * (u + ep)) @ vv.abs() + u * out[b, g].abs() + tiny * (1 + vv.abs().sum(0))
            w[b, h, :n] = p.sum(0)
            bw[b, h, :n] = (p * ep).sum(0) + 1e-37
    return out, bound, w, bw


def evict(weights, lengths, budget, sink, recent, cap):
    """Kept indices per (sequence, head), as lists."""
    B, K = weights.shape[:2]
    w = weights.double().cpu()
    rows = []
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        for h in range(K):
            if n <= budget:
                rows.append(list(range(n)))
                continue
            mid = list(range(min(sink, n), max(min(sink, n), n - recent)))
            x = w[b, h]
            mid.sort(key=lambda t: (-(float(x[t]) if x[t] == x[t] else float('-inf')), bool(x[t] != x[t]), t))
            stay = set(range(sink)) | set(range(n - recent, n)) | set(mid[:budget - sink - recent])
            rows.append(sorted(stay))
    return rows
