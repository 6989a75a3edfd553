"""Token sequences: rotary positions, attention under masks, paged key / value caches (csrc/rope.hip, masked_attn.hip, paged_attn.hip,
paged_evict.hip), for float32, float16 and bfloat16.

Beside the frame attention of this package (one bank of fp32 tokens per clip, sine positions, the oldest frames dropped first) these
are the forms a model over sequences of uneven length needs, in the order it calls them:

    freqs = rope_freqs(rot, ...)                         once: the turning frequencies, stretched for long contexts
    q, k = rope(q, k, pos, freqs)                        training / whole prompts, with gradients
    out = masked_attention(q, k, v, causal=True, ...)    documents, prefix, cap, distance bias; with gradients
    q = rope_append(q, k, v, pos, freqs, slots, k_pages, v_pages)      serving: turned keys and values into their cache places
    out = paged_attention(q, k_pages, v_pages, table, lengths, weights=w)   one new token per sequence, collecting attention weight
    kept, lengths, w, key_pos = paged_evict(k_pages, v_pages, table, lengths, w, new_table, budget=...)   thinning by that weight

Everything runs on the tensors' device and its current stream, allocates through torch only (hipGraph-capturable) and never waits for
the device.  A CPU tensor or a shape the kernels do not take raises AotHipError; there is no fallback."""
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

import aot_hip
from aot_hip import AotHipError


def rope_freqs(rot, base=10000.0, stretch=1.0, trained=4096, low=1.0, high=32.0, device=None):
    """Turning frequencies of the first `rot` elements of a head, float64 [rot / 2] in radians a position: base^(-2j / rot).
    stretch > 1 serves contexts that many times the `trained` length: a frequency that turns less than `low` times within the trained length is
    divided by stretch, one that turns more than `high` times is kept, those between are blended linearly in their number of turns."""
    if rot < 2 or rot % 2:
        raise AotHipError('rope_freqs: rot must be even and positive (got %d)' % rot)
    if stretch < 1.0 or not high > low:
        raise AotHipError('rope_freqs: stretch must be at least 1 and high above low')
    f = float(base) ** (-torch.arange(rot // 2, dtype=torch.float64) * 2.0 / rot)
    if stretch > 1.0:
        keep = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / stretch)
    return f if device is None else f.to(device)


class _Rope(Function):
    @staticmethod
    def forward(ctx, q, k, pos, freqs, interleaved, mscale):
        ctx.save_for_backward(pos, freqs)
        ctx.more = (interleaved, mscale)
        return aot_hip.rope(q, k, pos, freqs, interleaved, mscale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        pos, freqs = ctx.saved_tensors
        need_q, need_k = ctx.needs_input_grad[:2]
        if need_q and need_k:
            dq, dk = aot_hip.rope(dq, dk, pos, freqs, *ctx.more, inverse=True)
        elif need_q:
            dq, dk = aot_hip.rope(dq, None, pos, freqs, *ctx.more, inverse=True)[0], None
        elif need_k:
            dq, dk = None, aot_hip.rope(dk, None, pos, freqs, *ctx.more, inverse=True)[0]
        return dq, dk, None, None, None, None


def rope(q, k, pos, freqs, interleaved=False, mscale=1.0):
    """Rotary positions, differentiable in q and k.  q [B, S, H, D], k [B, S, Hk, D] or None (then one tensor is returned); pos int32 [B, S] or
    [S]; freqs float64 [rot / 2] (rope_freqs): the first rot elements of every head turn by pos * freqs, in pairs (j, j + rot / 2), or
    (2j, 2j + 1) if interleaved, and are multiplied by mscale; the others pass.  freqs has no gradient."""
    if freqs.requires_grad and torch.is_grad_enabled():
        raise AotHipError('rope: freqs have no gradient; pass freqs.detach()')
    if pos.dim() == 1:
        pos = pos.expand(q.shape[0], -1)
    if k is None:
        return _RopeOne.apply(q, pos, freqs, bool(interleaved), float(mscale))
    return _Rope.apply(q, k, pos, freqs, bool(interleaved), float(mscale))


class _RopeOne(Function):
    @staticmethod
    def forward(ctx, q, pos, freqs, interleaved, mscale):
        ctx.save_for_backward(pos, freqs)
        ctx.more = (interleaved, mscale)
        return aot_hip.rope(q, None, pos, freqs, interleaved, mscale)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dq):
        pos, freqs = ctx.saved_tensors
        return aot_hip.rope(dq, None, pos, freqs, *ctx.more, inverse=True)[0], None, None, None, None


class _MaskedAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, doc_q, doc_k, prefix, scale, causal, softcap):
        out, lse, res = aot_hip.attn_masked(q, k, v, scale, causal, softcap, slopes, doc_q, doc_k, prefix, residual=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, out, lse, res, slopes, doc_q, doc_k, prefix)
        ctx.more = (scale, causal, softcap)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, res, slopes, doc_q, doc_k, prefix = ctx.saved_tensors
        return aot_hip.attn_masked_bwd(dout, q, k, v, out, lse, res, *ctx.more, slopes, doc_q, doc_k, prefix) + (None,) * 7


def masked_attention(q, k, v, scale=None, causal=False, softcap=0.0, slopes=None, doc_q=None, doc_k=None, prefix=None):
    """Attention of q [B, Sq, H, D] over k / v [B, Sk, Hk, D] (H a multiple of Hk), differentiable in the three; out like q.

    Query i stands at place i + Sk - Sq among the keys.  scale (positive): 1 / sqrt(D) by default.  causal: keys up to the query's place.
    softcap: scores become softcap * tanh(score / softcap), 0: none.  slopes float32 [H]: slopes[h] * |distance| is taken off the score (no gradient).
    doc_q int32 [B, Sq], doc_k int32 [B, Sk]: a query sees the keys of its own document; a negative id is padding and sees nothing.
    prefix int32 [B]: under `causal`, keys before prefix[b] are seen by every query.  A query that sees nothing gives zeros and takes no
    gradient; what masked places hold never reaches a result."""
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise AotHipError('masked_attention: slopes have no gradient; pass slopes.detach()')
    return _MaskedAttention.apply(q, k, v, slopes, doc_q, doc_k, prefix, scale, bool(causal), float(softcap))


def _no_grad(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise AotHipError('%s is a serving call without gradients: run it under torch.no_grad()' % name)


def cache_slots(table, seq, pos, page):
    """Places of tokens in the pool: entry pos[n] of sequence seq[n] lies at table[seq, pos // page] * page + pos % page (int32).  -1 (rope_append
    writes nothing) for a padded token (pos or seq negative), for one outside the table, and for a page id that no int32 place can name."""
    B, n = table.shape
    if not table.numel():
        return torch.full(pos.shape, -1, dtype=torch.int32, device=pos.device)
    pos, seq = pos.long(), seq.long()
    ok = (pos >= 0) & (pos < n * page) & (seq >= 0) & (seq < B)
    slot = table[seq.clamp(0, B - 1), (pos // page).clamp(0, n - 1)].long() * page + pos.remainder(page)
    return torch.where(ok & (slot >= 0) & (slot <= 0x7fffffff), slot, -1).to(torch.int32)


def rope_append(q, k, v, pos, freqs, slots, k_pages, v_pages, interleaved=False, mscale=1.0):
    """Turns the new tokens' q [N, H, D] (or None) and k [N, Hk, D] by pos int32 [N], writes the turned keys and v [N, Hk, D] to the places slots
    int32 [N] (cache_slots; negative: a padded token, nothing is written; a place named twice holds parts of either token) of k_pages / v_pages
    [pages, page, Hk, D], returns the turned q."""
    _no_grad('rope_append', q, k, v, freqs, k_pages, v_pages)
    return aot_hip.rope_append(q, k, v, pos, freqs, slots, k_pages, v_pages, bool(interleaved), float(mscale))


def paged_attention(q, k_pages, v_pages, table, lengths, scale=None, softcap=0.0, slopes=None, weights=None, key_pos=None, out=None):
    """One new token per sequence, q [B, H, D], over its lengths[b] cache entries (its own the last of them); out like q.

    table int32 [B, max_pages]: entry t of sequence b lies at place t % page of page table[b, t // page].  softcap, slopes as in
    masked_attention; the distance is between places in the cache, or between key_pos int32 [B, Hk, S] where entries were evicted.
    weights float32 [B, Hk, S]: every entry's probability, summed over the query heads that share the key head, is added in place."""
    _no_grad('paged_attention', q, k_pages, v_pages, slopes, weights)
    return aot_hip.paged_attn(q, k_pages, v_pages, table, lengths, scale, float(softcap), slopes, weights, key_pos, out)


def paged_evict(k_pages, v_pages, table, lengths, weights, new_table, budget, sink=0, recent=0, key_pos=None):
    """Thins every cache row to `budget` entries: the first `sink`, the last `recent`, and of the rest those that collected most weight
    (ties: the earlier).  The kept rows are copied, in order, into the pages of new_table int32 [B, new_pages] -- pages no sequence uses;
    the old ones stay as they are for whoever shares them.  Key heads choose for themselves.  Returns (kept int32 [B, Hk, budget]: old places,
    -1 behind the last; new lengths; new weights and new key_pos, moved along).  Ids of -1 in new_table copy nothing: such a sequence goes on with
    its old table row, length, weights and positions."""
    _no_grad('paged_evict', k_pages, v_pages, weights)
    return aot_hip.paged_evict(k_pages, v_pages, table, lengths, weights, new_table, budget, sink, recent, key_pos)
