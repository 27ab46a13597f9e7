"""NumPy restatement of the block-scaled cache operators (oracle; test infrastructure).

Written from the definitions in include/pa_b200.h, one scale block and one row
at a time in float64; nothing here is shared with the library. Caches are
``(pages, heads, page_size, D)`` arrays of element values (``hnd`` order): codes
before their scale in 8 bits, plain values in 16. The 8-bit roundings come from
the formats' definitions (``float_to_e4m3`` is pinned against PyTorch by the
CPU tests); attention is ``reference.py:139-162`` per sequence.
"""

from __future__ import annotations

import math

import numpy as np

from .kvcache import e4m3_to_float, float_to_e4m3

__all__ = ["append_reference", "decode_reference", "evict_reference", "need_scale", "round8"]

QMAX = {"e4m3": 448.0, "int8": 127.0}


def round8(x, fmt):
    """Nearest value of the 8-bit format (ties to even, saturating; int8 has no NaN)."""
    x = np.asarray(x, np.float64)
    if fmt == "e4m3":
        return e4m3_to_float(float_to_e4m3(np.clip(x, -1e6, 1e6)))  # infinities saturate, NaN stays
    return np.where(np.isnan(x), 0.0, np.clip(np.rint(np.nan_to_num(x, nan=0.0, posinf=1e30, neginf=-1e30)), -127, 127))


def need_scale(x, fmt):
    """Least power of two s with max finite |x| <= qmax * s, at least 2^-100."""
    x = np.abs(np.asarray(x, np.float64))
    x = x[np.isfinite(x)]
    top = float(x.max()) if x.size else 0.0
    s = 2.0 ** -100
    if top > QMAX[fmt] * s:
        s = 2.0 ** (math.frexp(top)[1] - 12)
        while QMAX[fmt] * s < top:
            s *= 2.0
    return s


def _where(row, b, page_size, table):
    if table is None:
        return b, row
    return int(table[b][row // page_size]), row % page_size


def _rescale(codes, scales, page, h, block, incoming, held, fmt):
    """Put ``incoming`` (row in page -> values) into a block that holds the rows ``held``."""
    need = need_scale(np.concatenate([np.ravel(v) for v in incoming.values()]), fmt)
    old = float(scales[page, h, block])
    new = max(need, old) if held else need
    if held and new != old:
        for r in held:
            codes[page, h, r] = round8(codes[page, h, r] * old / new, fmt)
    for r, v in incoming.items():
        codes[page, h, r] = round8(v / new, fmt)
    scales[page, h, block] = new


def append_reference(k_new, v_new, k, v, lens, new_lens, *, ks=None, vs=None, table=None, block=None,
                     fmt=None, weights=None, positions=None, start=None):
    """Append in place; ``k_new`` is (batch, T, heads, D). Returns the new lengths."""
    page_size = k.shape[2]
    for x, cache, scales in ((k_new, k, ks), (v_new, v, vs)):
        x = np.asarray(x, np.float64)
        for b in range(len(lens)):
            n, t = int(lens[b]), int(new_lens[b])
            for h in range(k.shape[1]):
                if fmt is None:
                    for i in range(t):
                        page, at = _where(n + i, b, page_size, table)
                        cache[page, h, at] = x[b, i, h]
                    continue
                r = n
                while r < n + t:
                    lo = r // block * block
                    end = min(n + t, lo + block)
                    page, _ = _where(r, b, page_size, table)
                    place = {q: _where(q, b, page_size, table)[1] for q in range(lo, end)}
                    _rescale(cache, scales, page, h, place[r] // block,
                             {place[q]: x[b, q - n, h] for q in range(r, end)},
                             [place[q] for q in range(lo, r)], fmt)
                    r = end
    for b in range(len(lens)):
        n, t = int(lens[b]), int(new_lens[b])
        if weights is not None:
            weights[b, :, n:n + t] = 0.0
        if positions is not None:
            positions[b, :, n:n + t] = (n if start is None else int(start[b])) + np.arange(t)
    return np.asarray(lens) + np.asarray(new_lens)


def decode_reference(q, k, v, lens, *, ks=None, vs=None, table=None, block=None, scale=None, weights=None):
    """Returns a dict: ``out``, ``lse``, ``weights`` and what error bounds are derived from:
    ``pv`` = sum_j p_j |v_j| per output element, ``mag`` = max_j scale * sum_d |q_d k_jd| per head
    and ``p`` per (sequence, head, row)."""
    q = np.asarray(q, np.float64)
    B, Hq, D = q.shape
    H, page_size = k.shape[1], k.shape[2]
    G = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, pv = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    lse, mag = np.full((B, Hq), -np.inf), np.zeros((B, Hq))
    w = None if weights is None else np.array(weights, np.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        rows = np.arange(n)
        page = np.full(n, b) if table is None else np.asarray(table)[b, rows // page_size]
        at = rows if table is None else rows % page_size
        for h in range(H):
            kb, vb = k[page, h, at].astype(np.float64), v[page, h, at].astype(np.float64)
            if ks is not None:
                kb = kb * ks[page, h, at // block].astype(np.float64)[:, None]
                vb = vb * vs[page, h, at // block].astype(np.float64)[:, None]
            for g in range(h * G, (h + 1) * G):
                s = scale * (kb @ q[b, g])
                m = s.max()
                e = np.exp(s - m)
                p = e / e.sum()
                out[b, g], pv[b, g] = p @ vb, p @ np.abs(vb)
                lse[b, g] = m + math.log(e.sum())
                mag[b, g] = abs(scale) * (np.abs(kb) @ np.abs(q[b, g])).max()
                if w is not None:
                    w[b, h, :n] += p
    return {"out": out, "lse": lse, "weights": w, "pv": pv, "mag": mag}


def evict_reference(k, v, lens, weights, budget, *, recent=0, sinks=0, positions=None, next_positions=None,
                    ks=None, vs=None, table=None, block=None, fmt=None):
    """Evict in place (caches, scales, weights, positions). Returns ``(new lengths, kept)``."""
    B, H = weights.shape[:2]
    page_size = k.shape[2]
    kept = np.full((B, H, budget), -1, np.int32)
    k0, v0 = k.copy(), v.copy()
    ks0, vs0 = (None, None) if ks is None else (ks.copy(), vs.copy())
    for b in range(B):
        n = int(lens[b])
        nxt = n if next_positions is None else int(next_positions[b])
        for h in range(H):
            kept[b, h, :min(n, budget)] = np.arange(min(n, budget))
            if n <= budget:
                continue
            pos = np.arange(n) if positions is None else positions[b, h, :n].astype(np.int64)

            def rank(r):
                if pos[r] >= nxt - recent or pos[r] < sinks:
                    return (0, 0.0, r)
                x = float(weights[b, h, r])
                return (2, 0.0, r) if math.isnan(x) else (1, -x, r)

            keep = set(sorted(range(n), key=rank)[:budget])
            holes = [r for r in range(budget) if r not in keep]
            moves = dict(zip(holes, [r for r in range(budget, n) if r in keep]))
            for dst, src in moves.items():
                kept[b, h, dst] = src
                weights[b, h, dst] = weights[b, h, src]
                if positions is not None:
                    positions[b, h, dst] = positions[b, h, src]
            for cache, c0, scales, s0 in ((k, k0, ks, ks0), (v, v0, vs, vs0)):
                def value(src):
                    page, at = _where(src, b, page_size, table)
                    x = c0[page, h, at].astype(np.float64)
                    return x if fmt is None else x * float(s0[page, h, at // block])

                if fmt is None:
                    for dst, src in moves.items():
                        page, at = _where(dst, b, page_size, table)
                        cache[page, h, at] = value(src)
                    continue
                for lo in sorted({dst // block * block for dst in moves}):
                    rows = range(lo, min(lo + block, budget))
                    place = {r: _where(r, b, page_size, table) for r in rows}
                    _rescale(cache, scales, place[lo][0], h, place[lo][1] // block,
                             {place[r][1]: value(moves[r]) for r in rows if r in moves},
                             [place[r][1] for r in rows if r not in moves], fmt)
    return np.minimum(np.asarray(lens), budget), kept
