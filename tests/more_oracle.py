"""Plain 64-bit forms of the 8-bit paged cache, windows with sinks, the reservation of pages and logit
adjustments (test infrastructure)."""
import math

import numpy as np

BLOCK = 32  # positions of a scale


def e4m3():
    """The values of the 256 codes: sign, four bits of exponent (bias 7), three of mantissa; 0x7F and 0xFF are NaN."""
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0)) * np.where(c & 128, -1.0, 1.0)
    v[[127, 255]] = np.nan
    return v


CODES = e4m3()


def step(v):
    """The distance of the codes around |v| <= 448."""
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6)))
    return 2.0 ** (e - 3)


def encode(v):
    """The code nearest to each finite value of at most 448 in magnitude, ties to the even mantissa; NaN's is 0x7F."""
    v = np.asarray(v, np.float64)
    s = step(np.where(np.isnan(v), 0, v))
    r = np.rint(np.abs(np.where(np.isnan(v), 0, v)) / s) * s  # np.rint: ties to even, as the steps are the codes'
    c = np.searchsorted(CODES[:127], r)
    return np.where(np.isnan(v), 0x7F, c | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def exponent(top):
    """e of the least scale 2^e that takes `top` to at most 448, from -32 to 31."""
    if not top > 0:
        return -32
    m, e = math.frexp(top)  # 448 = 0.875 * 2^9
    return max(-32, min(31, e - 9 if m <= 0.875 else e - 8))


def k8_at(tok, dim, d):
    return (((tok // 32) * (d // 32) + dim // 32) * 1024 + dim % 32 // 8 * 256 + tok % 16 * 16 + tok % 32 // 16 * 8
            + dim % 8)


def v8_at(tok, dim, d):
    return (((tok // 32) * (d // 32) + dim // 32) * 1024 + tok % 16 // 4 * 256 + dim % 16 * 16 + dim % 32 // 16 * 8
            + tok % 32 // 16 * 4 + tok % 4)


def page_bytes(hkv, page, d):
    return hkv * page * d + -(-hkv * (page // BLOCK) * 4 // 128) * 128


def places8(table, positions, hkv, page, d, where):
    """Bytes [position][kv head][dim] of the codes in a pool."""
    pos = np.asarray(positions)
    base = np.asarray(table, np.int64)[pos // page] * page_bytes(hkv, page, d)
    return (base[:, None, None] + (np.arange(hkv) * page * d)[None, :, None]
            + where((pos % page)[:, None, None], np.arange(d)[None, None, :], d))


def scales_at(table, positions, hkv, page, d):
    """Indexes [position][kv head] of the scales in a pool of fp32."""
    pos = np.asarray(positions)
    base = np.asarray(table, np.int64)[pos // page] * page_bytes(hkv, page, d) + hkv * page * d
    return base[:, None] // 4 + np.arange(hkv)[None] * (page // BLOCK) + (pos % page // BLOCK)[:, None]


def visible(pos, window, sinks):
    """The positions that a row at `pos` attends to."""
    first = max(0, pos - window + 1) if window else 0
    return np.concatenate([np.arange(min(sinks if window else 0, first)), np.arange(first, pos + 1)])


def attend(q, k, v, keys, scale):
    """One row: q [hq][d] over the rows `keys` of k, v [positions][hkv][d]."""
    hq, hkv = q.shape[0], k.shape[1]
    out = np.zeros(q.shape)
    for h in range(hq):
        kk, vv = k[keys, h // (hq // hkv)].astype(np.float64), v[keys, h // (hq // hkv)].astype(np.float64)
        s = kk @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        out[h] = (p / p.sum()) @ vv
    return out


def pages_in_use(length, rows, window, sinks, page):
    """The pages that hold a position of the new rows, or one that the row at `length` sees."""
    first = max(0, length - window + 1) if window else 0
    return [i for i in range(-(-(length + rows) // page))
            if (i + 1) * page > first or (window and i * page < sinks)]


def reserve(tables, refs, lengths, counts, tokens, window, sinks, page, max_tokens):
    """(tables, refs, starts, slots, whether rows were left out, whether positions are lost) after the step."""
    tables, refs = tables.copy(), refs.copy()
    n, width = tables.shape
    starts, slots = np.full(n, -1, np.int32), np.full((n, tokens), -1, np.int64)
    limit = min(max_tokens, width * page)
    rows, lacks, bad, lost = [], [], False, False
    for s in range(n):
        p, c = int(lengths[s]), tokens if counts is None else int(counts[s])
        want = min(c, tokens) if p >= 0 and c > 0 else 0
        r = min(want, max(0, limit - p))
        bad |= want > 0 and (c > tokens or r < want)
        rows.append(r)
        use = set(pages_in_use(min(p, limit), r, window, sinks, page)) if p >= 0 else set()
        for i in range(width):
            e = int(tables[s, i])
            has = 0 <= e < refs.size
            if has and i not in use:
                refs[e] -= 1
            if not has or i not in use:
                tables[s, i] = -1
        lacks.append(sorted(i for i in use if tables[s, i] < 0))
    free = [int(p) for p in np.nonzero(refs == 0)[0]]
    asked = taken = 0
    for s in range(n):
        p = int(lengths[s])
        if any(i * page < p for i in lacks[s]):
            lost = True
            continue
        asked += len(lacks[s])
        if rows[s] < 1 or (lacks[s] and asked > len(free)):
            continue
        for i in lacks[s]:
            tables[s, i] = free[taken]
            refs[free[taken]] = 1
            taken += 1
        starts[s] = p
        for j in range(rows[s]):
            slots[s, j] = int(tables[s, (p + j) // page]) * page + (p + j) % page
    return tables, refs, starts, slots, bad, lost


def adjust(logits, counts, history, said, drafts, repetition, frequency, presence, bias_ids, biases, masks, out):
    """logits [n][t][v] under the rules, `out` where a row is not there; and |what was added| for its rounding."""
    n, t, v = logits.shape
    y, size = out.astype(np.float64).copy(), np.zeros((n, t, v))
    for s in range(n):
        for j in range(t if counts is None else min(t, int(counts[s]))):
            row = logits[s, j].astype(np.float64)
            big = np.abs(row)
            ids = np.zeros(0, np.int64)
            if history is not None:
                ids = history[s][:history.shape[1] if said is None else min(max(int(said[s]), 0), history.shape[1])]
            if drafts is not None:
                ids = np.concatenate([ids, drafts[s, :j]])
            ids, times = np.unique(ids[(ids >= 0) & (ids < v)].astype(np.int64), return_counts=True)
            r = 1.0 if repetition is None else float(repetition[s])
            f = 0.0 if frequency is None else float(frequency[s])
            p = 0.0 if presence is None else float(presence[s])
            with np.errstate(invalid="ignore", over="ignore"):
                old = row[ids]
                old = np.where(old > 0, old / r, old * r)
                row[ids] = old - p - f * times
                big[ids] = np.maximum(np.abs(old) + abs(p) + np.abs(f * times), big[ids])
                if bias_ids is not None:
                    for i, b in zip(bias_ids[s], biases[s]):
                        if 0 <= i < v:
                            row[i] += float(b)
                            big[i] += abs(float(b))
            if masks is not None:
                row[np.unpackbits(masks[s, j].view(np.uint8), bitorder="little")[:v] == 0] = -np.inf
            y[s, j], size[s, j] = row, big
    return y, size
