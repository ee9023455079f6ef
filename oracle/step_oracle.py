"""NumPy oracle of the serving-step operators, in 64 bits and from their definitions
(include/flash_engine_c.h): the step plan, the QKV append, the page boxes, and decode
attention over selected pages. Loops over requests, tokens and pages; for small sizes."""
import math

import numpy as np

MIN_EXP = -120


def plan(ctx, new, tables, ring, head, count, bs, max_tokens, finished=None):
    """Returns a dict; tables and ring are copied first."""
    S, width = tables.shape
    nb = len(ring)
    tables, old_ring, out_ring = tables.copy(), ring.copy(), ring.copy()
    old_tables = tables.copy()
    pushed = 0
    ctx = [max(0, int(c)) for c in ctx]
    for s in range(S):
        if finished is not None and finished[s]:
            for j in range(min(-(-ctx[s] // bs), width)):
                if count + pushed < nb:
                    out_ring[(head + count + pushed) % nb] = old_tables[s, j]
                pushed += 1
            ctx[s] = 0
    taken = tokens = served = 0
    lens = list(ctx)
    cu, pos, slots = [0], [], []
    open_ = True
    for s in range(S):
        n = max(0, int(new[s]))
        have = -(-ctx[s] // bs)
        need = -(-(ctx[s] + n) // bs) - have
        if tokens + n > max_tokens or taken + need > count or ctx[s] + n > width * bs:
            open_ = False
        if open_:
            served += 1
            for j in range(need):
                tables[s, have + j] = old_ring[(head + taken + j) % nb]
            for i in range(n):
                p = ctx[s] + i
                pos.append(p)
                slots.append(int(tables[s, p // bs]) * bs + p % bs)
            taken += need
            tokens += n
            lens[s] += n
        cu.append(tokens)
    pad = max_tokens - tokens
    return {"context_lens": np.array(lens, np.int32), "cu_seqlens": np.array(cu, np.int32),
            "positions": np.array(pos + [-1] * pad, np.int32),
            "slots": np.array(slots + [-1] * pad, np.int64), "tables": tables, "ring": out_ring,
            "state": np.array([(head + taken) % nb, min(nb, count - taken + pushed), served,
                               tokens], np.int32)}


def norm_rotate(x, w, eps, pos, cos, sin, interleaved):
    """x [n, d] float64 of tokens at pos [n]; w [d] or None; cos/sin [p, r/2] or None."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if cos is None:
        return x
    r = 2 * cos.shape[1]
    y = x.copy()
    c, s = np.asarray(cos, np.float64)[pos], np.asarray(sin, np.float64)[pos]
    i0, i1 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2),
                                                                    slice(r // 2, r))
    y[:, i0] = x[:, i0] * c - x[:, i1] * s
    y[:, i1] = x[:, i0] * s + x[:, i1] * c
    return y


def qkv_append(qkv, H, Hkv, d, kc, vc, pos, slots, bs, qw=None, kw=None, eps=1e-6, cos=None,
               sin=None, interleaved=True):
    """Queries [T, H, d] and new caches (flat layout [blocks, Hkv, bs, d], float64)."""
    T = qkv.shape[0]
    x = np.asarray(qkv, np.float64).reshape(T, H + 2 * Hkv, d)
    kc, vc = np.array(kc, np.float64), np.array(vc, np.float64)
    q = np.zeros((T, H, d))
    for t in range(T):
        p = int(pos[t])
        if p < 0 or (cos is not None and p >= cos.shape[0]):
            continue
        q[t] = norm_rotate(x[t, :H], qw, eps, [p] * H, cos, sin, interleaved)
        b, o = divmod(int(slots[t]), bs)
        if slots[t] < 0 or b >= kc.shape[0]:
            continue
        kc[b, :, o] = norm_rotate(x[t, H:H + Hkv], kw, eps, [p] * Hkv, cos, sin, interleaved)
        vc[b, :, o] = x[t, H + Hkv:]
    return q, kc, vc


def exponent(amax):
    """Smallest e >= MIN_EXP with amax <= 127 * 2^e, by search."""
    if amax == 0:
        return -7
    e = math.frexp(amax)[1] - 9
    while amax > 127 * 2.0 ** e:
        e += 1
    return max(e, MIN_EXP)


def boxes(k):
    """int8 values [n, Hkv, 2, d] and scales [n, Hkv] of pages [n, Hkv, bs, d]."""
    n, Hkv, bs, d = k.shape
    v, s = np.zeros((n, Hkv, 2, d), np.int8), np.zeros((n, Hkv), np.float32)
    for i in range(n):
        for h in range(Hkv):
            x = np.asarray(k[i, h], np.float64)
            if not np.isfinite(x).all():
                s[i, h] = np.inf
                continue
            e = exponent(np.abs(x).max())
            v[i, h, 0] = np.ceil(x.max(0) / 2.0 ** e)
            v[i, h, 1] = np.floor(x.min(0) / 2.0 ** e)
            s[i, h] = 2.0 ** e
    return v, s


def select(q, values, scales, table, ctx, bs, num_pages, first=1, last=1):
    """Chosen pages of one (sequence, KV head): q [G, d], table [width]."""
    P = -(-int(ctx) // bs)
    if P <= num_pages:
        return list(range(P))
    ints, unit = [], []
    for g in range(q.shape[0]):
        x = np.asarray(q[g], np.float64)
        if not np.isfinite(x).all():
            ints.append(None)
            unit.append(None)
            continue
        e = exponent(np.abs(x).max())
        ints.append(np.rint(x / 2.0 ** e).astype(np.int64))
        unit.append(e)
    score = []
    for j in range(P):
        b = int(table[j])
        if j < first or j >= P - last:
            score.append((1, 0.0))
            continue
        if np.isinf(scales[b]) or any(i is None for i in ints):
            score.append((0, math.inf))
            continue
        hi, lo = values[b, 0].astype(np.int64), values[b, 1].astype(np.int64)
        best = max(float(np.where(i > 0, i * hi, i * lo).sum()) * 2.0 ** u
                   for i, u in zip(ints, unit))
        score.append((0, best * float(scales[b])))
    order = sorted(range(P), key=lambda j: (-score[j][0], -score[j][1], j))
    return sorted(order[:num_pages])


def sparse_attention(q, kc, vc, values, scales, tables, ctx, bs, num_pages, first=1, last=1,
                     scale=None):
    """out [S, H, d] float64 and the chosen pages [S, Hkv, num_pages] (-1 padded)."""
    S, H, d = q.shape
    Hkv = kc.shape[1]
    G = H // Hkv
    out, sel = np.zeros((S, H, d)), np.full((S, Hkv, num_pages), -1, np.int32)
    scale = scale or 1 / math.sqrt(d)
    for s in range(S):
        for h in range(Hkv):
            qs = np.asarray(q[s, h * G:(h + 1) * G], np.float64)
            pages = select(qs, values[:, h], scales[:, h], tables[s], ctx[s], bs, num_pages,
                           first, last)
            sel[s, h, :len(pages)] = pages
            if not pages:
                continue
            at = [(int(tables[s, j]), o) for j in pages for o in range(bs) if j * bs + o < ctx[s]]
            b, o = np.array(at).T
            k, v = np.asarray(kc[b, h, o], np.float64), np.asarray(vc[b, h, o], np.float64)
            x = qs @ k.T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            out[s, h * G:(h + 1) * G] = (p / p.sum(-1, keepdims=True)) @ v
    return out, sel
