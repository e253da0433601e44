"""Plain 64-bit forms of the paged operators and of draft verification (test infrastructure)."""
import numpy as np

LOWEST = -3.4028234663852886e38


def k_at(tok, dim, d, e):
    return ((tok // 16) * (d // e) + dim // e) * 16 * e + (tok % 16) * e + dim % e


def v_at(tok, dim, d, e):
    g = 4 * e
    return ((tok // g) * (d // 16) + dim // 16) * 64 * e + ((tok % 16) // 4 * 16 + dim % 16) * e + tok % g // 16 * 4 + tok % 4


def places(table, positions, hkv, page, d, e, where):
    """Pool indexes [position][kv head][dim]."""
    pos = np.asarray(positions)
    base = np.asarray(table, np.int64)[pos // page] * (hkv * page * d)
    return (base[:, None, None] + (np.arange(hkv) * page * d)[None, :, None]
            + where((pos % page)[:, None, None], np.arange(d)[None, None, :], d, e))


def rope(x, pos, inv, factor=1.0):
    """Rotate-half over the first 2 len(inv) dims of x [rows][heads][d]."""
    if inv is None:
        return x.astype(np.float64)
    ang = np.asarray(pos, np.float64)[:, None] * inv[None, :].astype(np.float64)
    c, s = np.cos(ang)[:, None, :] * factor, np.sin(ang)[:, None, :] * factor
    h = inv.size
    a, b = x[..., :h].astype(np.float64), x[..., h:2 * h].astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def attend(q, k, v, pos, window, scale, there=None):
    """One row: q [hq][d] over k, v [positions][hkv][d], positions 0 .. pos; `there`: which have a page."""
    hq, hkv = q.shape[0], k.shape[1]
    first = max(0, pos - window + 1) if window else 0
    keys = np.arange(first, pos + 1)
    if there is not None:
        keys = keys[there[keys]]
    out = np.zeros(q.shape)
    if keys.size == 0:
        return out
    for h in range(hq):
        kk, vv = k[keys, h // (hq // hkv)].astype(np.float64), v[keys, h // (hq // hkv)].astype(np.float64)
        s = kk @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        out[h] = (p / p.sum()) @ vv
    return out


def softmax(row, temp):
    """Probabilities and whether the row has an entry that takes part."""
    x = np.asarray(row, np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        part = np.asarray(row, np.float32) > np.float32(LOWEST)
    p = np.zeros_like(x)
    if not part.any():
        return p, False
    m = x[part].max()
    d = np.where(x[part] == m, 0.0, x[part] - m if np.isfinite(m) else -np.inf)
    p[part] = np.exp(d / temp)
    return p / p.sum(), True


def pick(w, u):
    c = np.cumsum(w)
    if not c[-1] > 0:
        return -1
    over = np.nonzero((c > float(u) * c[-1]) & (w > 0))[0]
    return int(over[0]) if over.size else int(np.nonzero(w > 0)[0][-1])


def verify(logits, drafts, counts, uniforms, temp, draft_logits=None):
    """(accepted, tokens) with -7 where a result stays as it was."""
    n, t, v = logits.shape
    accepted, ids = np.full(n, -7, np.int32), np.full((n, t), -7, np.int32)
    for s in range(n):
        c = t if counts is None else min(int(counts[s]), t)
        if c < 1:
            continue
        ids[s], accepted[s] = -1, 0
        for j in range(c):
            x = int(drafts[s, j]) if j + 1 < c else None
            inside = x is not None and 0 <= x < v
            if temp == 0:
                row = logits[s, j]
                with np.errstate(invalid="ignore"):
                    part = row > np.float32(LOWEST)
                best = int(np.argmax(np.where(part, row, -np.inf))) if part.any() else -1
                stands, token = inside and best == x, best
            else:
                p, some = softmax(logits[s, j], max(temp, 1e-6))
                q = np.zeros(v)
                if x is not None and draft_logits is not None:
                    q, _ = softmax(draft_logits[s, j], max(temp, 1e-6))
                elif inside:
                    q[x] = 1.0
                stands = inside and float(uniforms[s, j]) * q[x] < p[x]
                if not stands:
                    token = pick(np.maximum(p - q, 0), uniforms[s, t - 1])
                    if token < 0:
                        token = pick(p, uniforms[s, t - 1])
            if not stands:
                ids[s, j] = token
                break
            ids[s, j] = x
            accepted[s] += 1
    return accepted, ids
