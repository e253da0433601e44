"""Operators of a server's step over paged caches, as cases to be timed.

    listed()             the named cases
    draw(rng)            one more case of the ranges that they stand for
    prepare(case, seed)  what a program has in hand before the call
    run(state)           one pass: the plain form, or with `own` the library's entry points
    work(case)           the bytes and operations that a pass cannot do without
    exact(case, seed)    the same results in 64 bits, from the definitions

The operators, in the order in which a step uses them:

    reserve    the sequences' page tables, first positions and slots, from their lengths
    append     new rows rotated and stored in a cache of 8-bit values
    attention  of the new rows over the pages: of an 8-bit cache, and with a sliding window whose
               first tokens stay visible, over every type of cache
    adjust     penalties, biases and masks on the logits, before a token is picked

Head shapes and vocabularies are those of the package's own workloads (three-llm_amd/weights.py).

A pool of 16 or 32-bit values holds pages [page][kv head][page tokens x head_dim]; within a page, 16-byte pieces
of E elements (8 of fp16, 4 of fp32) lie in the order
    K  [token / 16][dim / E][token % 16][dim % E]
    V  [token / (4 E)][dim / 16][token % 16 / 4][dim % 16][token % (4 E) / 16][token % 4]
A pool of 8-bit values (e4m3) holds pages of bytes: the codes [kv head][page tokens x head_dim] in the order
    K  [token / 32][dim / 32][dim % 32 / 8][token % 16][token % 32 / 16][dim % 8]
    V  [token / 32][dim / 32][token % 16 / 4][dim % 16][dim % 32 / 16][token % 32 / 16][token % 4]
and behind them the scales, fp32 [kv head][page tokens / 32], up to a multiple of 128 bytes.  A value is its
code times the scale of its 32 tokens: the least power of two from 2^-32 to 2^31 that takes the largest
magnitude to at most 448.  An append within 32 tokens keeps the larger of the scale that they have and the one
that its rows need; tokens before it that get a larger one are rounded again.
"""
import ctypes
import importlib.util
import json
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parents[1]

# (query heads, kv heads, head_dim, RoPE theta) of the package's workloads
HEADS = {"tiny": (4, 2, 64, 1e4), "qwen2.5-0.5b": (14, 2, 64, 1e6), "llama-3.2-1b": (32, 8, 64, 5e5),
         "llama-3.2-3b": (24, 8, 128, 5e5)}
DTYPE = {"f16": torch.float16, "f32": torch.float32}
SIZE = {"f8": 1, "f16": 2, "f32": 4}
F8 = torch.float8_e4m3fn
BLOCK = 32  # tokens of a scale


def listed():
    return [
        # A server's step over 64 chats with four drafts each, in a pool of which other programs hold a part.
        {"name": "reserve 64x5 @8192", "op": "reserve", "seqs": 64, "tokens": 5, "longest": 8192, "page": 64,
         "window": 0, "sinks": 0, "short": False},
        # Many chats of a model with a window, in a pool with few spare pages: those before the windows come back.
        {"name": "reserve 1024x1 @32768 w4096", "op": "reserve", "seqs": 1024, "tokens": 1, "longest": 32768,
         "page": 32, "window": 4096, "sinks": 64, "short": True},
        # The next token of a busy server's 64 chats, most within 32 tokens that have a scale.
        {"name": "append f8 llama-1b 64x1", "op": "append", "heads": "llama-3.2-1b", "seqs": 64, "tokens": 1,
         "longest": 700, "page": 32, "kv": "f8", "window": 0, "sinks": 0, "idle": 3},
        # Two prompts' chunks at once, the second behind a cached prefix.
        {"name": "append f8 llama-3b 2x2048", "op": "append", "heads": "llama-3.2-3b", "seqs": 2, "tokens": 2048,
         "longest": 1000, "page": 128, "kv": "f8", "window": 0, "sinks": 0, "idle": 0},
        # Attention of one chat's next token over an 8-bit cache: the smallest call.
        {"name": "attention f8 qwen 1x1 @300", "op": "attention", "heads": "qwen2.5-0.5b", "seqs": 1, "tokens": 1,
         "longest": 300, "page": 64, "kv": "f8", "out": "f32", "window": 0, "sinks": 0, "idle": 0},
        # The busy server's step: 64 chats of very different lengths.
        {"name": "attention f8 llama-1b 64x1 @8192", "op": "attention", "heads": "llama-3.2-1b", "seqs": 64,
         "tokens": 1, "longest": 8192, "page": 64, "kv": "f8", "out": "f16", "window": 0, "sinks": 0, "idle": 3},
        # Four drafted tokens and the one before them, for 16 chats.
        {"name": "attention f8 llama-3b 16x5 @2500", "op": "attention", "heads": "llama-3.2-3b", "seqs": 16,
         "tokens": 5, "longest": 2500, "page": 128, "kv": "f8", "out": "f16", "window": 0, "sinks": 0, "idle": 0},
        # One endless chat: four first tokens and the last 4096.
        {"name": "sinks f16 llama-3b 1x1 w4096", "op": "attention", "heads": "llama-3.2-3b", "seqs": 1, "tokens": 1,
         "longest": 32768, "page": 256, "kv": "f16", "out": "f16", "window": 4096, "sinks": 4, "idle": 0},
        # Many endless chats with a system prompt that stays, the pages between given back.
        {"name": "sinks f8 llama-1b 64x1 w1024", "op": "attention", "heads": "llama-3.2-1b", "seqs": 64, "tokens": 1,
         "longest": 8192, "page": 64, "kv": "f8", "out": "f16", "window": 1024, "sinks": 100, "idle": 1},
        # Prompts' chunks with a window that is shorter than they are.
        {"name": "sinks f16 qwen 4x500 w300", "op": "attention", "heads": "qwen2.5-0.5b", "seqs": 4, "tokens": 500,
         "longest": 1500, "page": 64, "kv": "f16", "out": "f16", "window": 300, "sinks": 4, "idle": 0},
        # One chat with four drafts and penalties over what it has said so far.
        {"name": "adjust 1x5 151936", "op": "adjust", "seqs": 1, "tokens": 5, "vocab": 151936, "history": 900,
         "biases": 0, "masked": False, "idle": 0},
        # 64 chats with everything: penalties over long histories, biases, a grammar's masks.
        {"name": "adjust 64x1 128256 masked", "op": "adjust", "seqs": 64, "tokens": 1, "vocab": 128256,
         "history": 4096, "biases": 32, "masked": True, "idle": 2},
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["reserve", "append", "attention", "attention", "sinks", "sinks", "adjust"])
    if op == "reserve":
        window = rng.choice([0, _log(rng, 1, 8192)])
        return {"op": op, "seqs": _log(rng, 1, 1024), "tokens": rng.choice([1, rng.randint(2, 16), _log(rng, 17, 512)]),
                "longest": _log(rng, 1, 32768), "page": rng.choice([32, 64, 128, 256]), "window": window,
                "sinks": rng.choice([0, rng.randint(1, 200)]) if window else 0, "short": rng.choice([False, True])}
    seqs = _log(rng, 1, 64)
    idle = rng.choice([0, 0, 1]) if seqs > 1 else 0
    if op == "adjust":
        tokens = rng.choice([1, rng.randint(2, 9)])
        seqs = min(seqs, 64 // tokens)
        return {"op": op, "seqs": seqs, "tokens": tokens, "vocab": _log(rng, 4096, 128256),
                "history": _log(rng, 1, 4096), "biases": rng.choice([0, rng.randint(1, 300)]),
                "masked": rng.choice([False, True]), "idle": min(idle, seqs - 1)}
    case = {"op": "attention" if op == "sinks" else op, "heads": rng.choice(sorted(HEADS)),
            "page": rng.choice([32, 64, 128, 256]), "kv": "f8", "window": 0, "sinks": 0}
    if op == "append":
        case["tokens"] = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 2048)])
        case["longest"] = _log(rng, 1, 1000)
        case["seqs"] = min(seqs, max(1, 2500 // case["tokens"]))
    else:
        case["tokens"] = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, 400)])
        case["seqs"] = seqs = min(seqs, max(1, 600 // case["tokens"]))
        if op == "sinks":
            case.update(kv=rng.choice(["f8", "f16", "f32"]), window=_log(rng, 1, 3000), sinks=_log(rng, 1, 200))
        _, hkv, d, _ = HEADS[case["heads"]]
        most = 160000000 // (seqs * 2 * hkv * d * SIZE[case["kv"]])  # positions, at the bytes of the largest listed
        case["longest"] = max(1, min(_log(rng, 1, 32768), most))
        case["out"] = rng.choice(["f16", "f32"])
    return dict(case, idle=min(idle, case["seqs"] - 1))


# ------------------------------------------------------------------ inputs --

_kept = {}


def _plan(case):
    """(starts, counts) of the sequences: the first position of this step's rows and how many are new.  They are
    the case's own, so that its work is known; an idle slot starts at -1."""
    rng = random.Random(case["seqs"] * 1000003 + case["tokens"] * 7919 + case["longest"])
    n, t = case["seqs"], case["tokens"]
    starts = [case["longest"] - 1 if s == 0 else _log(rng, max(1, case["longest"] // 16), case["longest"]) - 1
              for s in range(n)]
    counts = [t if s == 0 else rng.randint((t + 1) // 2, t) for s in range(n)]
    for s in range(case["idle"]):
        starts[n - 1 - s * (n // 8 + 1)] = -1
    return starts, counts


def _first(case, start):
    """The first position of the window of a row at `start`."""
    return max(0, start - case["window"] + 1) if case["window"] else 0


def _in_use(case, start, rows):
    """The pages that a sequence needs for rows at start, start + 1, ...: (those of its sinks end, the others
    begin, and end)."""
    page = case["page"]
    end = -(-(start + rows) // page)
    first = min(_first(case, start) // page, end)
    return min(-(-case["sinks"] // page), first), first, end


def _gen(*key):
    g = torch.Generator(device="cuda")
    s = 0x9E3779B9
    for v in key:
        s = (s * 1000003 + int(v) + 1) % (1 << 62)
    g.manual_seed(s)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype) * std


def _inv_freq(d, theta):
    return (theta ** (-np.arange(0, d, 2, dtype=np.float64) / d)).astype(np.float32)


def _page_bytes(hkv, page, d):
    """Bytes of a page's codes in an 8-bit pool, and of the page."""
    codes = hkv * page * d
    return codes, codes + -(-hkv * (page // BLOCK) * 4 // 128) * 128


def _pool8(g, pages, hkv, page, d):
    """A pool as earlier steps left it: values of about unit scale under scales of 2^-8 to 2^-6."""
    codes, size = _page_bytes(hkv, page, d)
    pool = torch.zeros(pages, size, dtype=torch.uint8, device="cuda")
    pool[:, :codes] = _normal(g, pages, codes, std=100.0).clamp(-448, 448).to(F8).view(torch.uint8)
    _scales(pool, hkv, page, d).copy_(
        torch.exp2(torch.randint(-8, -5, (pages, hkv, page // BLOCK), generator=g, device="cuda").float()))
    return pool


def _inputs(case, seed):
    """The sequences' tables over a shuffled pool (-1 where a sequence has no page), the pool as earlier steps left
    it (unit scale, also past the sequences' ends), and this step's rows."""
    hq, hkv, d, theta = HEADS[case["heads"]]
    n, t, page = case["seqs"], case["tokens"], case["page"]
    starts, counts = _plan(case)
    used = [_in_use(case, s, c) if s >= 0 else (0, 0, 0) for s, c in zip(starts, counts)]
    width = max(e for _, _, e in used)
    pages = sum(a + e - b for a, b, e in used) + 3
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, (a, b, e) in enumerate(used):
        for lo, hi in ((0, a), (b, e)):
            tables[s, lo:hi] = order[at:at + hi - lo]
            at += hi - lo
    if case["kv"] == "f8":
        k, v = (_pool8(_gen(seed, i), pages, hkv, page, d) for i in (2, 3))
    else:
        k, v = (_normal(_gen(seed, i), pages, hkv, page * d, dtype=DTYPE[case["kv"]]) for i in (2, 3))
    rows = (hq + 2 * hkv) * d if case["op"] == "append" else hq * d
    x = _normal(_gen(seed, 4), n * t, rows)
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"k": k, "v": v, "tables": tables, "starts": torch.tensor(starts, **i32),
            "counts": torch.tensor(counts, **i32), "x": x}


def _pool_plan(case):
    """What a server has before it reserves, on the host: lengths, counts, tables over pages 0, 1, ... (every second
    sequence without a window shares a prefix with the one before), what holds each page, the pages of the pool."""
    key = json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True)
    if key in _kept:
        return _kept[key]
    n, t, page = case["seqs"], case["tokens"], case["page"]
    rng = random.Random(n * 1000003 + t * 7919 + case["longest"])
    width = -(-(case["longest"] + t) // page)
    lengths, counts = np.zeros(n, np.int32), np.zeros(n, np.int32)
    tables = np.full((n, width), -1, np.int32)
    refs, at, need = [], 0, 0
    before = 0
    for s in range(n):
        kind = rng.choice(["goes on"] * 13 + ["new", "ended", "waits"]) if s else "goes on"
        length = case["longest"] if s == 0 else _log(rng, max(1, case["longest"] // 16), case["longest"])
        said = min(length, rng.randint(1, t))  # the step before: its rows that stood
        had = min(t, length - said + t) if kind != "new" else 0
        used = _in_use(case, length - said, min(had, width * page - (length - said))) if kind != "new" else (0, 0, 0)
        ids = list(range(0, used[0])) + list(range(used[1], used[2]))
        shared = 0
        if s % 2 and not case["window"] and before > 1 and len(ids) > 1:
            shared = min(before, len(ids)) // 2
            tables[s, :shared] = tables[s - 1, :shared]
            for p in tables[s, :shared]:
                refs[p] += 1
        for i in ids[shared:]:
            tables[s, i] = at
            refs.append(1)
            at += 1
        before = len(ids) if not case["window"] else 0
        lengths[s] = -1 if kind == "ended" else 0 if kind == "new" else length
        counts[s] = 0 if kind == "waits" else t if s == 0 else rng.randint((t + 1) // 2, t)
        if kind != "ended":
            rows = max(0, min(int(counts[s]), width * page - int(lengths[s])))
            a, b, e = _in_use(case, int(lengths[s]), rows)
            have = set(i for i in range(width) if tables[s, i] >= 0)
            need += sum(i not in have for i in list(range(a)) + list(range(b, e)))
    spare = need // 3 if case["short"] else need + 8
    others = 1 + at // 8  # pages that hold what is no sequence's
    refs += [1] * others + [0] * spare
    _kept[key] = lengths, counts, tables, np.array(refs, np.int32)
    return _kept[key]


def _reserve_inputs(case, seed):
    lengths, counts, tables, refs = _pool_plan(case)
    order = torch.randperm(refs.size, generator=_gen(seed, 1), device="cuda")
    t = torch.from_numpy(tables).cuda()
    r = torch.empty(refs.size, dtype=torch.int32, device="cuda")
    r[order] = torch.from_numpy(refs).cuda()
    t = torch.where(t >= 0, order[t.clamp_min(0).long()].to(torch.int32), t)
    return {"lengths": torch.from_numpy(lengths).cuda(), "counts": torch.from_numpy(counts).cuda(), "tables": t,
            "refs": r}


def _adjust_inputs(case, seed):
    """Logits of broad scale; histories in which few tokens are many (u^3), most of them full; every chat with
    settings of its own; masks of three kinds: a grammar's fixed words, its lists, its free text."""
    n, t, v = case["seqs"], case["tokens"], case["vocab"]
    i32 = dict(dtype=torch.int32, device="cuda")
    d = {"logits": _normal(_gen(seed, 1), n * t, v, std=3.0)}
    rng = random.Random(n * 1000003 + t * 7919 + v)
    counts = [t if s == 0 else rng.randint((t + 1) // 2, t) for s in range(n)]
    for s in range(case["idle"]):
        counts[n - 1 - s * (n // 8 + 1)] = 0
    said = [case["history"] if s % 3 else _log(rng, 1, case["history"]) for s in range(n)]
    d["counts"], d["said"] = torch.tensor(counts, **i32), torch.tensor(said, **i32)

    def tokens(key, *shape):
        return (torch.rand(*shape, generator=_gen(seed, key), device="cuda") ** 3 * v).to(torch.int32).clamp(max=v - 1)

    d["past"] = tokens(2, n, case["history"])
    if t > 1:
        d["drafts"] = tokens(3, n, t - 1)
    u = torch.rand(3, n, generator=_gen(seed, 4), device="cuda")
    d["repetition"], d["frequency"], d["presence"] = (1 + 0.5 * u[0]).contiguous(), u[1] - 0.2, u[2] - 0.2
    if case["biases"]:
        d["bias_ids"] = torch.randint(-1, v, (n, case["biases"]), generator=_gen(seed, 5), device="cuda").to(torch.int32)
        d["biases_of"] = _normal(_gen(seed, 6), n, case["biases"], std=5.0)
    if case["masked"]:
        share = torch.tensor([0.002, 0.5, 0.97], device="cuda")[torch.arange(n * t, device="cuda") % 3]
        bits = torch.rand(n * t, -(-v // 32) * 32, generator=_gen(seed, 7), device="cuda") < share[:, None]
        place = torch.arange(32, device="cuda")
        words = (bits.view(n * t, -1, 32).long() << place).sum(-1)
        d["masks"] = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return d


def prepare(case, seed):
    s = dict(case)
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "reserve":
        s.update(_reserve_inputs(case, seed))
        n, t = case["seqs"], case["tokens"]
        s["out_tables"], s["out_refs"] = torch.zeros_like(s["tables"]), torch.zeros_like(s["refs"])
        s["starts"], s["slots"] = torch.zeros(n, **i32), torch.zeros(n, t, dtype=torch.int64, device="cuda")
    elif case["op"] == "adjust":
        s.update(_adjust_inputs(case, seed))
        s["out"] = torch.zeros_like(s["logits"])
    else:
        s.update(_inputs(case, seed))
        hq, hkv, d, theta = HEADS[case["heads"]]
        dt = torch.float32 if case["op"] == "append" else DTYPE[case["out"]]
        s["y"] = torch.zeros(case["seqs"], case["tokens"], hq * d, dtype=dt, device="cuda")
        s["inv_freq"] = torch.from_numpy(_inv_freq(d, theta)).cuda()
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------- the plain forms --

def _k_view(pool, page, d):
    e = 16 // pool.element_size()
    return pool.view(pool.shape[0], pool.shape[1], page // 16, d // e, 16, e)


def _v_view(pool, page, d):
    s = 4 // pool.element_size()
    return pool.view(pool.shape[0], pool.shape[1], page // (16 * s), d // 16, 4, 16, s, 4)


def _k8_view(pool, hkv, page, d):
    return pool[:, :hkv * page * d].view(pool.shape[0], hkv, page // BLOCK, d // 32, 4, 16, 2, 8)


def _v8_view(pool, hkv, page, d):
    return pool[:, :hkv * page * d].view(pool.shape[0], hkv, page // BLOCK, d // 32, 4, 16, 2, 2, 4)


def _scales(pool, hkv, page, d):
    codes, n = hkv * page * d, hkv * (page // BLOCK)
    return pool[:, codes:codes + 4 * n].view(torch.float32).view(pool.shape[0], hkv, page // BLOCK)


def _positions(s):
    """Positions of the rows [n][t] and which rows are there."""
    j = torch.arange(s["tokens"], device="cuda")
    pos = s["starts"].long()[:, None] + j
    return pos, (s["starts"] >= 0)[:, None] & (j < s["counts"][:, None])


def _needed(top):
    """The scale of values up to `top`."""
    m, e = torch.frexp(top)  # 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.ldexp(torch.ones_like(top), torch.where(top > 0, e.clamp(-32, 31), -32))


def _append(s):
    hq, hkv, d, _ = HEADS[s["heads"]]
    n, t, page = s["seqs"], s["tokens"], s["page"]
    pos, live = _positions(s)
    x = s["x"].view(n, t, hq + 2 * hkv, d)
    angle = pos[:, :, None, None].double() * s["inv_freq"].double()
    c, sn = angle.cos().float(), angle.sin().float()
    a, b = x[:, :, :hq + hkv, :d // 2], x[:, :, :hq + hkv, d // 2:]
    rot = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    s["y"].copy_(torch.where(live[:, :, None], rot[:, :, :hq].reshape(n, t, hq * d), s["y"]))
    # the blocks of 32 tokens that the rows lie in, from the first row's on
    many = (t + BLOCK - 2) // BLOCK + 1
    start = s["starts"].long()
    p0 = (start[:, None] // BLOCK + torch.arange(many, device="cuda")) * BLOCK
    there = (p0 <= start[:, None] + s["counts"][:, None] - 1) & live[:, :1]
    at = s["tables"].long().gather(1, (p0 // page).clamp(0, s["tables"].shape[1] - 1))
    held = (start[:, None] - p0).clamp_min(0)  # tokens that the block has already: of the first one only
    of = (pos // BLOCK - start[:, None] // BLOCK)  # the block of a row
    seq, blk = there.nonzero(as_tuple=True)
    bseq, row = live.nonzero(as_tuple=True)
    page_of, in_page = at[seq, blk], p0[seq, blk] % page // BLOCK
    kp = at[bseq, of[bseq, row]]
    tok = pos[bseq, row] % page
    for pool, rows in ((s["k"], rot[:, :, hq:]), (s["v"], x[:, :, hq + hkv:])):
        is_k = pool is s["k"]
        codes, scales = (_k8_view if is_k else _v8_view)(pool, hkv, page, d), _scales(pool, hkv, page, d)
        top = torch.zeros(n, many, hkv, device="cuda")
        size = torch.where(live[:, :, None], rows.abs().amax(-1), 0.0)
        top.scatter_reduce_(1, of.clamp(0, many - 1)[:, :, None].expand(n, t, hkv), size, "amax")
        scale = _needed(top)[seq, blk]
        old = scales[page_of, :, in_page]
        mid = held[seq, blk] > 0
        scale = torch.where(mid[:, None], torch.maximum(scale, old), scale)
        # what the block has already, under its new scale
        m = mid.nonzero()[:, 0]
        had = codes[page_of[m], :, in_page[m]]
        i, sub = torch.arange(16, device="cuda"), torch.arange(2, device="cuda")
        if is_k:  # [..][16][2][8]
            token = (i[:, None] + 16 * sub)[:, :, None]
        else:  # [4][16][2][2][4]
            token = (4 * i[:4, None, None] + 16 * sub[:, None] + i[:4])[:, None, None]
        keep = token < held[seq, blk][m].view(-1, *[1] * (had.dim() - 1))
        ratio = (old / scale)[m].view(m.shape[0], hkv, *[1] * (had.dim() - 2))
        again = (had.view(F8).float() * ratio).to(F8).view(torch.uint8)
        codes[page_of[m], :, in_page[m]] = torch.where(keep, again, had)
        scales[page_of, :, in_page] = scale
        of_row = torch.zeros(n, many, hkv, device="cuda")
        of_row[seq, blk] = scale
        new = (rows[bseq, row] / of_row[bseq, of[bseq, row]][:, :, None]).to(F8).view(torch.uint8)
        if is_k:
            codes[kp, :, tok // 32, :, :, tok % 16, tok % 32 // 16] = new.view(-1, hkv, d // 32, 4, 8)
        else:
            codes[kp, :, tok // 32, :, tok % 16 // 4, :, :, tok % 32 // 16, tok % 4] = (
                new.view(-1, hkv, d // 32, 2, 16).transpose(-1, -2))
    return _appended(s)


def _appended(s):
    """The rotated queries and the pools: codes as the 8-bit numbers that they are, and their scales."""
    _, hkv, d, _ = HEADS[s["heads"]]
    at = (hkv, s["page"], d)
    return {"q": s["y"], "k": s["k"][:, :hkv * s["page"] * d].view(F8), "k_scales": _scales(s["k"], *at),
            "v": s["v"][:, :hkv * s["page"] * d].view(F8), "v_scales": _scales(s["v"], *at)}


def _rows_of(s, pool, at, tok, is_k):
    """Rows [n][keys][kv head][d] of tokens of pages, in 32 bits."""
    _, hkv, d, _ = HEADS[s["heads"]]
    page, shape = s["page"], (*at.shape, hkv, d)
    if s["kv"] == "f8":
        if is_k:
            c = _k8_view(pool, hkv, page, d)[at, :, tok // 32, :, :, tok % 16, tok % 32 // 16]
        else:
            c = _v8_view(pool, hkv, page, d)[at, :, tok // 32, :, tok % 16 // 4, :, :, tok % 32 // 16, tok % 4]
            c = c.transpose(-1, -2).contiguous()
        return c.view(F8).float().view(shape) * _scales(pool, hkv, page, d)[at, :, tok // BLOCK][..., None]
    if is_k:
        return _k_view(pool, page, d)[at, :, tok // 16, :, tok % 16].float().view(shape)
    sub = 4 // pool.element_size()
    return _v_view(pool, page, d)[at, :, tok // (16 * sub), :, tok % 16 // 4, :, tok % (16 * sub) // 16,
                                  tok % 4].float().view(shape)


def _attention(s):
    hq, hkv, d, _ = HEADS[s["heads"]]
    n, t, page, window, sinks = s["seqs"], s["tokens"], s["page"], s["window"], s["sinks"]
    g = hq // hkv
    pos, live = _positions(s)
    end = s["tables"].shape[1] * page
    if window and window + t + sinks < end:  # the sinks before the first window, and the windows
        first = (s["starts"].long() - window + 1).clamp_min(0)[:, None]
        key = torch.arange(sinks, device="cuda")[None]
        key = torch.where(key < first, key, end)
        key = torch.cat([key, first + torch.arange(window + t - 1, device="cuda")], 1)
    else:
        key = torch.arange(end, device="cuda").expand(n, end)
    at = s["tables"].long().gather(1, (key // page).clamp_max(s["tables"].shape[1] - 1)).clamp_min(0)
    keys = key.shape[1]
    k = _rows_of(s, s["k"], at, key % page, True).transpose(1, 2)
    v = _rows_of(s, s["v"], at, key % page, False).transpose(1, 2).contiguous()
    q = s["x"].view(n, t, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, t * g, d)
    score = (q @ k.transpose(2, 3).contiguous()).view(n, hkv, t, g, keys) * d ** -0.5
    key = key[:, None]
    seen = (key <= pos[:, :, None]) & live[:, :, None]
    if window:
        seen &= (key > pos[:, :, None] - window) | (key < sinks)
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    y = (p.view(n, hkv, t * g, keys) @ v).view(n, hkv, t, g, d) / p.sum(-1, keepdim=True).clamp_min(1e-38)
    y = y.permute(0, 2, 1, 3, 4).reshape(n, t, hq * d).to(s["y"].dtype)
    s["y"].copy_(torch.where(live[:, :, None], y, s["y"]))
    return s["y"]


def _reserve(s):
    page, window, sinks = s["page"], s["window"], s["sinks"]
    tables, refs = s["tables"], s["refs"]
    n, width = tables.shape
    pages = refs.shape[0]
    length = s["lengths"].long()
    rows = torch.where(length >= 0, s["counts"].long().clamp(0, s["tokens"]), 0)
    rows = torch.minimum(rows, (width * page - length).clamp_min(0))
    i = torch.arange(width, device="cuda") * page
    first = (length - window + 1).clamp_min(0)[:, None] if window else torch.zeros_like(length)[:, None]
    used = (i < (length + rows)[:, None]) & ((i + page > first) | (i < sinks))
    has = (tables >= 0) & (tables < pages)
    gone, lost = has & ~used, used & ~has & (i < length[:, None])
    need = used & ~has & (i >= length[:, None]) & ~lost.any(1, keepdim=True)
    wants = need.sum(1)
    refs = refs.clone()
    back = tables[gone].long()
    refs.index_add_(0, back, torch.full_like(back, -1, dtype=torch.int32))
    free = refs == 0
    served = (rows > 0) & ~lost.any(1) & ((wants == 0) | (wants.cumsum(0) <= free.sum()))
    take = need & served[:, None]
    order = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")  # the free pages, lowest first
    order[torch.where(free, free.cumsum(0) - 1, pages)] = torch.arange(pages, device="cuda")
    rank = (take.view(-1).cumsum(0) - 1).view(n, width)
    new = order[rank.clamp(0, pages)]
    refs.index_add_(0, new[take], torch.ones_like(new[take], dtype=torch.int32))
    out = torch.where(take, new, torch.where(has & used, tables.long(), -1))
    s["out_tables"].copy_(out)
    s["out_refs"].copy_(refs)
    s["starts"].copy_(torch.where(served, length, -1))
    j = torch.arange(s["tokens"], device="cuda")
    pos = length[:, None] + j
    slot = out.gather(1, (pos // page).clamp(0, width - 1)) * page + pos % page
    s["slots"].copy_(torch.where(served[:, None] & (j < rows[:, None]), slot, -1))
    return _reserved(s)


def _reserved(s):
    return {"tables": s["out_tables"], "refs": s["out_refs"], "starts": s["starts"], "slots": s["slots"]}


def _adjust(s):
    n, t, v = s["seqs"], s["tokens"], s["vocab"]
    times = torch.zeros(n, v + 1, device="cuda")
    there = torch.arange(s["history"], device="cuda") < s["said"][:, None]
    times.scatter_add_(1, torch.where(there, s["past"].long(), v), there.float())
    times = times[:, None, :v].expand(n, t, v)
    if t > 1:
        more = torch.zeros(n, t, v, device="cuda")
        more[:, 1:].scatter_(2, s["drafts"].long()[:, :, None], 1.0)
        times = times + more.cumsum(1)
    each = {k: s[k].double()[:, None, None] for k in ("repetition", "frequency", "presence")}
    x = s["logits"].view(n, t, v).double()
    y = torch.where(x > 0, x / each["repetition"], x * each["repetition"])
    y = torch.where(times > 0, y - each["presence"] - each["frequency"] * times, x)
    if s["biases"]:
        bias = torch.zeros(n, v + 1, dtype=torch.float64, device="cuda")
        ids = s["bias_ids"].long()
        bias.scatter_add_(1, torch.where(ids >= 0, ids, v), s["biases_of"].double())
        y = y + bias[:, None, :v]
    if s["masked"]:
        i = torch.arange(v, device="cuda")
        bit = s["masks"].view(n, t, -1)[:, :, i // 32] >> (i % 32).to(torch.int32) & 1
        y = y.masked_fill(bit == 0, -math.inf)
    live = (torch.arange(t, device="cuda") < s["counts"][:, None])[:, :, None]
    s["out"].copy_(torch.where(live, y, s["out"].view(n, t, v)).view(n * t, v))
    return s["out"]


# ------------------------------------------------------ the library's calls --

def _tlm():
    if "tlm" not in _kept:
        if "three_llm_amd" not in sys.modules:
            pkg = ROOT / "three-llm_amd"
            spec = importlib.util.spec_from_file_location("three_llm_amd", pkg / "__init__.py",
                                                          submodule_search_locations=[str(pkg)])
            mod = importlib.util.module_from_spec(spec)
            sys.modules["three_llm_amd"] = mod
            spec.loader.exec_module(mod)
        _kept["tlm"] = sys.modules["three_llm_amd"].tlm
        _kept["ctx"] = _kept["tlm"].Context(0)
    return _kept["tlm"], _kept["ctx"]


class Dev:
    """A torch tensor as the device buffer that the entry points take."""

    def __init__(self, t):
        self.t = t
        self.ptr = ctypes.c_void_p(t.data_ptr())


def _paged(s):
    """The program's handle for a model and page size, kept for all its sequences."""
    tlm, ctx = _tlm()
    hq, hkv, d, theta = HEADS[s.get("heads", "tiny")]
    key = (s.get("heads"), s["page"], s["window"], s["sinks"], s.get("kv"))
    if key not in _kept:
        fmt = {"f8": tlm.FMT_F8, "f16": tlm.FMT_F16, "f32": tlm.FMT_F32}[s.get("kv", "f16")]
        _kept[key] = tlm.Paged(ctx, hq, hkv, d, max_tokens=1 << 16, page_tokens=s["page"],
                               inv_freq=_inv_freq(d, theta), sliding_window=s["window"], kv_fmt=fmt)
        if s["sinks"]:
            _kept[key].set_sinks(s["sinks"])
    return _kept[key]


def _bind(s):
    """What a program keeps from step to step: its buffers' addresses and the call's arguments that name them."""
    tlm, ctx = _tlm()
    d = s["dev"] = {k: Dev(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["op"] == "adjust":
        s["rules"] = tlm.logit_rules(
            d["logits"], s["seqs"], s["tokens"], s["vocab"], out=d["out"], counts=d["counts"], history=d["past"],
            history_width=s["history"], history_counts=d["said"], drafts=d.get("drafts"),
            repetition=d["repetition"], frequency=d["frequency"], presence=d["presence"],
            bias_ids=d.get("bias_ids"), biases=d.get("biases_of"), bias_width=s["biases"], masks=d.get("masks"))
        return
    s["paged"] = _paged(s)
    if s["op"] == "reserve":
        s["request"] = s["paged"].request(
            d["lengths"], d["tables"], s["tables"].shape[1], d["refs"], s["refs"].shape[0], d["starts"], s["seqs"],
            s["tokens"], counts=d["counts"], slots=d["slots"], out_tables=d["out_tables"], out_refs=d["out_refs"])
        return
    s["batch"] = s["paged"].batch(d["k"], d["v"], s["k"].shape[0], d["tables"], s["tables"].shape[1], d["starts"],
                                  s["seqs"], s["tokens"], counts=d["counts"])
    if s["op"] == "append":
        s["views"] = _appended(s)  # of its own buffers


def _own(s):
    tlm, ctx = _tlm()
    if "dev" not in s:
        _bind(s)
    d = s["dev"]
    if s["op"] == "reserve":
        s["paged"].reserve(s["request"])
        return _reserved(s)
    if s["op"] == "append":
        s["paged"].append(s["batch"], d["x"], d["y"])
        return s["views"]
    if s["op"] == "attention":
        s["paged"].attention(s["batch"], d["x"], d["y"], {"f16": tlm.FMT_F16, "f32": tlm.FMT_F32}[s["out"]])
        return s["y"]
    tlm.adjust_logits(ctx, s["rules"])
    return s["out"]


def run(s):
    if own:
        return _own(s)
    return {"reserve": _reserve, "append": _append, "attention": _attention, "adjust": _adjust}[s["op"]](s)


# ------------------------------------------------------------------- figures --

def work(case):
    n, t = case["seqs"], case["tokens"]
    if case["op"] == "reserve":
        _, _, tables, refs = _pool_plan(case)
        return {"bytes": 8 * tables.size + 8 * refs.size + 12 * n + 8 * n * t, "flops": 0}
    if case["op"] == "adjust":
        rows = (n - case["idle"]) * t
        size = 8 * case["vocab"] + (case["vocab"] // 8 if case["masked"] else 0)
        return {"bytes": rows * size + n * (4 * case["history"] + 8 * case["biases"]), "flops": 0}
    hq, hkv, d, _ = HEADS[case["heads"]]
    starts, counts = _plan(case)
    live = [(s, c) for s, c in zip(starts, counts) if s >= 0]
    rows, size = sum(c for _, c in live), SIZE[case["kv"]]
    if case["op"] == "append":
        return {"bytes": rows * d * ((hq + 2 * hkv) * 4 + 2 * hkv * size + hq * 4), "flops": 6.0 * rows * (hq + hkv) * d}
    keys = sum(s + c - _first(case, s) + min(case["sinks"], _first(case, s)) for s, c in live)
    seen = sum(p + 1 - _first(case, p) + min(case["sinks"], _first(case, p)) for s, c in live for p in range(s, s + c))
    scales = 2 * hkv * 4 * keys // BLOCK if case["kv"] == "f8" else 0
    return {"bytes": keys * 2 * hkv * d * size + scales + rows * hq * d * (4 + SIZE[case["out"]]),
            "flops": 4.0 * hq * d * seen}


# ------------------------------------------------------------------- 64 bits --

def _k_place(tok, dim, page, d, size):
    """Where element (token of the page, dim) of K lies in a page's head."""
    if size == 1:
        return ((tok // 32) * (d // 32) + dim // 32) * 1024 + dim % 32 // 8 * 256 + tok % 16 * 16 + tok % 32 // 16 * 8 + dim % 8
    e = 16 // size
    return ((tok // 16) * (d // e) + dim // e) * 16 * e + (tok % 16) * e + dim % e


def _v_place(tok, dim, page, d, size):
    if size == 1:
        return (((tok // 32) * (d // 32) + dim // 32) * 1024 + tok % 16 // 4 * 256 + dim % 16 * 16 + dim % 32 // 16 * 8
                + tok % 32 // 16 * 4 + tok % 4)
    e = 16 // size
    g = 4 * e
    return ((tok // g) * (d // 16) + dim // 16) * 64 * e + ((tok % 16) // 4 * 16 + dim % 16) * e + (tok % g) // 16 * 4 + tok % 4


def _places(case, x, s, pos, where):
    """Flat indexes [position][kv head][dim] into a pool, of positions of sequence s."""
    _, hkv, d, _ = HEADS[case["heads"]]
    page, size = case["page"], SIZE[case["kv"]]
    step = _page_bytes(hkv, page, d)[1] if size == 1 else hkv * page * d
    base = x["tables"][s].long()[pos // page] * step
    head = torch.arange(hkv, device="cuda") * (page * d)
    dim = torch.arange(d, device="cuda")
    return (base[:, None, None] + head[None, :, None]
            + where((pos % page)[:, None, None], dim[None, None, :], page, d, size))


def _e4m3():
    """The values of the 256 codes: sign, four bits of exponent (bias 7), three of mantissa."""
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0)) * np.where(c & 128, -1.0, 1.0)
    v[[127, 255]] = np.nan
    return torch.from_numpy(v).cuda()


def _scale_at(case, x, s, pos):
    """Flat indexes [position][kv head] of the scales in a pool of fp32."""
    _, hkv, d, _ = HEADS[case["heads"]]
    page = case["page"]
    codes, size = _page_bytes(hkv, page, d)
    base = (x["tables"][s].long()[pos // page] * size + codes) // 4
    return base[:, None] + torch.arange(hkv, device="cuda") * (page // BLOCK) + (pos % page // BLOCK)[:, None]


def _values(case, x, pool, s, pos, where):
    """Rows [position][kv head][dim] of sequence s in 64 bits."""
    at = _places(case, x, s, pos, where)
    if case["kv"] != "f8":
        return pool.view(-1)[at].double()
    return _e4m3()[pool.view(-1)[at].long()] * pool.view(torch.float32).view(-1)[_scale_at(case, x, s, pos)].double()[..., None]


def _exact_append(case, seed):
    hq, hkv, d, theta = HEADS[case["heads"]]
    n, t, page = case["seqs"], case["tokens"], case["page"]
    x = _inputs(case, seed)
    starts, counts = _plan(case)
    codes = hkv * page * d
    inv = torch.from_numpy(_inv_freq(d, theta)).cuda().double()
    rows = x["x"].view(n, t, hq + 2 * hkv, d)
    q = torch.zeros(n, t, hq * d, dtype=torch.float64, device="cuda")
    out = {"q": q}
    pools = {}
    for name in ("k", "v"):
        c = torch.zeros(x[name].shape, dtype=torch.float64, device="cuda")
        c[:, :codes] = _e4m3()[x[name][:, :codes].long()]
        pools[name] = c, x[name].view(torch.float32).double().clone()
    for s in range(n):
        p0, c = starts[s], counts[s]
        if p0 < 0:
            continue
        r = rows[s, :c].double()
        z = torch.complex(r[:, :hq + hkv, : d // 2], r[:, :hq + hkv, d // 2:])
        ang = torch.arange(p0, p0 + c, device="cuda").double()[:, None] * inv
        z = z * torch.polar(torch.ones_like(ang), ang)[:, None]
        z = torch.cat([z.real, z.imag], -1)
        q[s, :c] = z[:, :hq].reshape(c, hq * d)
        for name, new, where in (("k", z[:, hq:], _k_place), ("v", r[:, hq + hkv:], _v_place)):
            val, sc = pools[name]
            for b in range(p0 // BLOCK, (p0 + c - 1) // BLOCK + 1):
                lo, hi = max(p0, b * BLOCK), min(p0 + c, (b + 1) * BLOCK)
                top = new[lo - p0:hi - p0].abs().amax((0, 2)).cpu().numpy()
                want = np.array([2.0 ** min(31, max(-32, math.ceil(math.log2(v / 448)))) if v > 0 else 2.0 ** -32 for v in top])
                want = torch.from_numpy(want).cuda()
                at = _scale_at(case, x, s, torch.tensor([b * BLOCK], device="cuda"))[0]
                if lo > b * BLOCK:
                    was = sc.view(-1)[at]
                    want = torch.maximum(want, was)
                    old = _places(case, x, s, torch.arange(b * BLOCK, lo, device="cuda"), where)
                    val.view(-1)[old] *= (was / want)[None, :, None]
                sc.view(-1)[at] = want
                pos = torch.arange(lo, hi, device="cuda")
                val.view(-1)[_places(case, x, s, pos, where)] = new[lo - p0:hi - p0] / want[None, :, None]
    many = hkv * (page // BLOCK)
    for name in ("k", "v"):
        val, sc = pools[name]
        out[name] = val[:, :codes].contiguous()
        out[name + "_scales"] = sc[:, codes // 4:codes // 4 + many].reshape(-1, hkv, page // BLOCK)
    return out


def _exact_attention(case, seed):
    hq, hkv, d, _ = HEADS[case["heads"]]
    n, t, g = case["seqs"], case["tokens"], hq // hkv
    x = _inputs(case, seed)
    starts, counts = _plan(case)
    y = torch.zeros(n, t, hq * d, dtype=torch.float64, device="cuda")
    rows = x["x"].view(n, t, hq, d).double()
    for s in range(n):
        p0, c = starts[s], counts[s]
        if p0 < 0:
            continue
        first = _first(case, p0)
        pos = torch.cat([torch.arange(min(case["sinks"], first), device="cuda"),
                         torch.arange(first, p0 + c, device="cuda")])
        k = _values(case, x, x["k"], s, pos, _k_place).permute(1, 2, 0)  # [head][dim][position]
        v = _values(case, x, x["v"], s, pos, _v_place).permute(1, 0, 2)
        for j in range(0, c, 32):
            at = torch.arange(j, min(c, j + 32), device="cuda")
            w = rows[s, at].view(-1, hkv, g, d).permute(1, 0, 2, 3).reshape(hkv, -1, d) @ k.contiguous()
            w = w.view(hkv, at.shape[0], g, -1) / math.sqrt(d)
            here = p0 + at[:, None]
            seen = pos[None] <= here
            if case["window"]:
                seen &= (here - pos[None] < case["window"]) | (pos[None] < case["sinks"])
            w = torch.softmax(w.masked_fill(~seen[None, :, None], -math.inf), -1)
            o = w.view(hkv, -1, pos.shape[0]) @ v.contiguous()
            y[s, at] = o.view(hkv, -1, g, d).transpose(0, 1).reshape(-1, hq * d)
    return y


def _exact_reserve(case, seed):
    x = {k: v.cpu().numpy().copy() for k, v in _reserve_inputs(case, seed).items()}
    n, t, page, tables, refs = case["seqs"], case["tokens"], case["page"], x["tables"], x["refs"]
    width = tables.shape[1]
    starts, slots = np.full(n, -1, np.int32), np.full((n, t), -1, np.int64)
    rows = [max(0, min(int(c), t, width * page - int(p))) if p >= 0 else 0 for p, c in zip(x["lengths"], x["counts"])]
    kept = []
    for s in range(n):
        p = int(x["lengths"][s])
        keep = set()
        if p >= 0:
            a, b, e = _in_use(case, p, rows[s])
            keep = set(range(a)) | set(range(b, e))
        for i in range(width):
            if tables[s, i] >= 0 and i not in keep:
                refs[tables[s, i]] -= 1
                tables[s, i] = -1
        kept.append(sorted(i for i in keep if tables[s, i] < 0))
    free = [int(p) for p in np.nonzero(refs == 0)[0]]
    asked = taken = 0
    for s in range(n):
        p = int(x["lengths"][s])
        if any(i * page < p for i in kept[s]):
            continue
        asked += len(kept[s])
        if rows[s] < 1 or (kept[s] and asked > len(free)):
            continue
        for i in kept[s]:
            tables[s, i] = free[taken]
            refs[free[taken]] += 1
            taken += 1
        starts[s] = p
        for j in range(rows[s]):
            slots[s, j] = int(tables[s, (p + j) // page]) * page + (p + j) % page
    return {k: torch.from_numpy(v) for k, v in (("tables", tables), ("refs", refs), ("starts", starts), ("slots", slots))}


def _exact_adjust(case, seed):
    n, t, v = case["seqs"], case["tokens"], case["vocab"]
    x = {k: a.cpu().numpy() for k, a in _adjust_inputs(case, seed).items()}
    y = np.zeros((n, t, v))
    for s in range(n):
        for j in range(min(t, int(x["counts"][s]))):
            row = x["logits"][s * t + j].astype(np.float64)
            ids = x["past"][s, :x["said"][s]]
            if j:
                ids = np.concatenate([ids, x["drafts"][s, :j]])
            ids, times = np.unique(ids, return_counts=True)
            r, f, p = (float(x[k][s]) for k in ("repetition", "frequency", "presence"))
            old = row[ids]
            row[ids] = np.where(old > 0, old / r, old * r) - p - f * times
            for i in range(case["biases"]):
                if x["bias_ids"][s, i] >= 0:
                    row[x["bias_ids"][s, i]] += x["biases_of"][s, i]
            if case["masked"]:
                row[np.unpackbits(x["masks"][s * t + j].view(np.uint8), bitorder="little")[:v] == 0] = -np.inf
            y[s, j] = row
    return torch.from_numpy(y.reshape(n * t, v))


def exact(case, seed):
    return {"reserve": _exact_reserve, "append": _exact_append, "attention": _exact_attention,
            "adjust": _exact_adjust}[case["op"]](case, seed)
