"""Operators for serving many sequences at once from a paged cache, as cases to be timed.

    listed()             the named cases
    draw(rng)            one more case of the ranges that they stand for
    prepare(case, seed)  what a program has in hand before the call
    run(state)           one pass: the plain form, or with `own` the library's entry points
    work(case)           the bytes and operations that a pass cannot do without
    exact(case, seed)    the same results in 64 bits, from the definitions

Three operators: the rows of a step rotated and appended to the pages of their
sequences, attention of each sequence's new tokens over its pages, and the
verification of drafted tokens.  Head shapes and vocabularies are those of the
package's own workloads (three-llm_amd/weights.py).

A pool holds pages [page][kv head][page tokens x head_dim].  Within a page, 16-byte
pieces of E elements (8 of fp16, 4 of fp32) lie in the order
    K  [token / 16][dim / E][token % 16][dim % E]
    V  [token / (4 E)][dim / 16][token % 16 / 4][dim % 16][token % (4 E) / 16][token % 4]
"""
import ctypes
import importlib.util
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
SIZE = {"f16": 2, "f32": 4}


def listed():
    return [
        # One chat's next token on the smallest real model: launches and latency.
        {"name": "append qwen 1x1", "op": "append", "heads": "qwen2.5-0.5b", "seqs": 1, "tokens": 1, "longest": 300,
         "page": 64, "kv": "f16", "window": 0, "idle": 0},
        # A step of a busy server: one token of each of 64 chats, three slots idle.
        {"name": "append llama-1b 64x1", "op": "append", "heads": "llama-3.2-1b", "seqs": 64, "tokens": 1,
         "longest": 700, "page": 32, "kv": "f16", "window": 0, "idle": 3},
        # Two prompts' chunks at once, the second behind a cached prefix.
        {"name": "append llama-3b 2x2048", "op": "append", "heads": "llama-3.2-3b", "seqs": 2, "tokens": 2048,
         "longest": 1000, "page": 128, "kv": "f16", "window": 0, "idle": 0},
        # Attention of one chat's next token: the smallest call.
        {"name": "attention qwen 1x1 @300", "op": "attention", "heads": "qwen2.5-0.5b", "seqs": 1, "tokens": 1,
         "longest": 300, "page": 64, "kv": "f16", "out": "f32", "window": 0, "idle": 0},
        # The busy server's step: 64 chats of very different lengths.
        {"name": "attention llama-1b 64x1 @8192", "op": "attention", "heads": "llama-3.2-1b", "seqs": 64, "tokens": 1,
         "longest": 8192, "page": 64, "kv": "f16", "out": "f16", "window": 0, "idle": 3},
        # Four drafted tokens and the one before them, for 16 chats.
        {"name": "attention llama-3b 16x5 @2500", "op": "attention", "heads": "llama-3.2-3b", "seqs": 16, "tokens": 5,
         "longest": 2500, "page": 128, "kv": "f16", "out": "f16", "window": 0, "idle": 0},
        # One long document: the work lies along one cache.
        {"name": "attention llama-3b 1x1 @32768", "op": "attention", "heads": "llama-3.2-3b", "seqs": 1, "tokens": 1,
         "longest": 32768, "page": 256, "kv": "f16", "out": "f16", "window": 0, "idle": 0},
        # A sliding window over a 32-bit cache, pages before the window given back.
        {"name": "attention llama-1b 8x1 f32 w1000", "op": "attention", "heads": "llama-3.2-1b", "seqs": 8, "tokens": 1,
         "longest": 5000, "page": 32, "kv": "f32", "out": "f32", "window": 1000, "idle": 0},
        # One chat with four tokens that a lookup drafted (no draft probabilities).
        {"name": "verify 1x5 128256 lookup", "op": "verify", "seqs": 1, "tokens": 5, "vocab": 128256, "by": "lookup",
         "temperature": 0.8, "idle": 0},
        # 32 chats with drafts of a small model, whose logits come too.
        {"name": "verify 32x5 151936 model", "op": "verify", "seqs": 32, "tokens": 5, "vocab": 151936, "by": "model",
         "temperature": 0.8, "idle": 1},
        # No drafts: one token sampled for each of 64 chats.
        {"name": "verify 64x1 32000", "op": "verify", "seqs": 64, "tokens": 1, "vocab": 32000, "by": "lookup",
         "temperature": 1.0, "idle": 0},
        # Greedy decoding with eight drafted tokens.
        {"name": "verify 16x9 128256 greedy", "op": "verify", "seqs": 16, "tokens": 9, "vocab": 128256, "by": "lookup",
         "temperature": 0.0, "idle": 0},
    ]


def _log(rng, lo, hi):
    """A whole number, its logarithm uniform over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "verify"])
    seqs = _log(rng, 1, 64)
    idle = rng.choice([0, 0, 1]) if seqs > 1 else 0
    if op == "verify":
        tokens = rng.choice([1, rng.randint(2, 9)])
        return {"op": op, "seqs": min(seqs, 160 // tokens), "tokens": tokens, "vocab": _log(rng, 4096, 151936),
                "by": rng.choice(["lookup", "model"]), "temperature": rng.choice([0.0, 0.3, 0.8, 1.0]), "idle": idle}
    case = {"op": op, "heads": rng.choice(sorted(HEADS)), "seqs": seqs, "page": rng.choice([32, 64, 128, 256]),
            "kv": rng.choice(["f16", "f16", "f32"]), "window": rng.choice([0, 0, 512, rng.randint(1, 3000)]),
            "idle": idle}
    if op == "append":
        case["tokens"] = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 2048)])
        case["longest"] = _log(rng, 1, 1000)
        case["seqs"] = min(seqs, max(1, 2500 // case["tokens"]))
    else:
        case["tokens"] = rng.choice([1, 1, rng.randint(2, 16)])
        _, hkv, d, _ = HEADS[case["heads"]]
        most = 320000000 // (seqs * 2 * hkv * d * SIZE[case["kv"]])  # positions, at the bytes of the largest listed
        case["longest"] = min(_log(rng, 1, 32768), most)
        case["out"] = rng.choice(["f16", "f32"])
    return dict(case, idle=min(idle, case["seqs"] - 1))


# ------------------------------------------------------------------ inputs --

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
    """The first position that a row at `start` attends to."""
    return max(0, start - case["window"] + 1) if case["window"] else 0


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


def _pages(case):
    """Pages of each sequence's table, those in use, and the pool's pages."""
    starts, counts = _plan(case)
    page = case["page"]
    width = max(-(-(s + c) // page) for s, c in zip(starts, counts) if s >= 0)
    used = [(_first(case, s) // page, -(-(s + c) // page)) if s >= 0 else (0, 0) for s, c in zip(starts, counts)]
    return width, used, sum(b - a for a, b in used) + 3


def _inputs(case, seed):
    """The sequences' tables over a shuffled pool (-1 where a sequence has no page), the pool as earlier steps left
    it (unit scale, also past the sequences' ends), and this step's rows."""
    hq, hkv, d, theta = HEADS[case["heads"]]
    n, t = case["seqs"], case["tokens"]
    starts, counts = _plan(case)
    width, used, pages = _pages(case)
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, (a, b) in enumerate(used):
        tables[s, a:b] = order[at:at + b - a]
        at += b - a
    dt = DTYPE[case["kv"]]
    k = _normal(_gen(seed, 2), pages, hkv, case["page"] * d, dtype=dt)
    v = _normal(_gen(seed, 3), pages, hkv, case["page"] * d, dtype=dt)
    rows = (hq + 2 * hkv) * d if case["op"] == "append" else hq * d
    x = _normal(_gen(seed, 4), n * t, rows)
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"k": k, "v": v, "tables": tables, "starts": torch.tensor(starts, **i32),
            "counts": torch.tensor(counts, **i32), "x": x}


def _verify_inputs(case, seed):
    """Target logits of unit-to-broad scale, the drafts and (from a draft model) the logits they were drawn from."""
    n, t, v, temp = case["seqs"], case["tokens"], case["vocab"], case["temperature"]
    logits = _normal(_gen(seed, 1), n * t, v, std=2.5)
    d = {"logits": logits, "uniforms": torch.rand(n, t, generator=_gen(seed, 2), device="cuda")}
    rng = random.Random(seed)
    counts = [t if s == 0 else rng.randint((t + 1) // 2, t) for s in range(n)]
    for s in range(case["idle"]):
        counts[n - 1 - s] = 0
    d["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    if t > 1:
        about = logits.view(n, t, v)[:, :-1]
        if case["by"] == "model":
            d["draft_logits"] = (about + _normal(_gen(seed, 3), n, t - 1, v, std=0.6)).contiguous()
            about = d["draft_logits"]
        # a draw at the temperature (of what is likeliest, where it is 0 and for a lookup) by perturbed scores
        u = torch.rand(n, t - 1, v, generator=_gen(seed, 4), device="cuda").clamp_min(1e-20)
        scale = max(temp, 0.3) if case["by"] == "model" else 0.2
        d["drafts"] = (about / scale - torch.log(-torch.log(u))).argmax(-1).to(torch.int32)
    return d


def prepare(case, seed):
    s = dict(case)
    if case["op"] == "verify":
        s.update(_verify_inputs(case, seed))
        i32 = dict(dtype=torch.int32, device="cuda")
        s["accepted"] = torch.zeros(case["seqs"], **i32)
        s["ids"] = torch.zeros(case["seqs"], case["tokens"], **i32)
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


def _positions(s):
    """Positions of the rows [n][t] and which rows are there."""
    j = torch.arange(s["tokens"], device="cuda")
    pos = s["starts"].long()[:, None] + j
    return pos, (s["starts"] >= 0)[:, None] & (j < s["counts"][:, None])


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
    # the pages of the rows that are there, and the token in the page
    seq, row = live.nonzero(as_tuple=True)
    p = pos[seq, row]
    at, tok = s["tables"][seq, p // page].long(), p % page
    kv, vv = _k_view(s["k"], page, d), _v_view(s["v"], page, d)
    e, sub = kv.shape[-1], vv.shape[-2]
    m = seq.shape[0]
    kv[at, :, tok // 16, :, tok % 16, :] = rot[seq, row, hq:].reshape(m, hkv, d // e, e).to(kv.dtype)
    vv[at, :, tok // (16 * sub), :, tok % 16 // 4, :, tok % (16 * sub) // 16, tok % 4] = (
        x[seq, row, hq + hkv:].reshape(m, hkv, d // 16, 16).to(vv.dtype))
    return {"q": s["y"], "k": s["k"], "v": s["v"]}


def _attention(s):
    hq, hkv, d, _ = HEADS[s["heads"]]
    n, t, page = s["seqs"], s["tokens"], s["page"]
    g = hq // hkv
    pos, live = _positions(s)
    at = s["tables"].long().clamp_min(0)
    keys = at.shape[1] * page
    k = _k_view(s["k"], page, d)[at].permute(0, 2, 1, 3, 5, 4, 6).reshape(n, hkv, keys, d).float()
    v = _v_view(s["v"], page, d)[at].permute(0, 2, 1, 3, 7, 5, 8, 4, 6).reshape(n, hkv, keys, d).float()
    q = s["x"].view(n, t, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, t * g, d)
    score = (q @ k.transpose(2, 3).contiguous()).view(n, hkv, t, g, keys) * d ** -0.5
    key = torch.arange(keys, device="cuda")
    seen = (key <= pos[:, :, None]) & live[:, :, None]
    if s["window"]:
        seen &= key > pos[:, :, None] - s["window"]
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    y = (p.view(n, hkv, t * g, keys) @ v).view(n, hkv, t, g, d) / p.sum(-1, keepdim=True).clamp_min(1e-38)
    y = y.permute(0, 2, 1, 3, 4).reshape(n, t, hq * d).to(s["y"].dtype)
    s["y"].copy_(torch.where(live[:, :, None], y, s["y"]))
    return s["y"]


def _verify(s):
    n, t, v, temp = s["seqs"], s["tokens"], s["vocab"], s["temperature"]
    logits, counts = s["logits"].view(n, t, v), s["counts"].long()
    j = torch.arange(t, device="cuda")
    real = j[:-1] < (counts - 1)[:, None]  # drafts that are there
    if temp == 0:
        best = logits.argmax(-1)
        ok = best[:, :-1] == s["drafts"] if t > 1 else real
        taken = (ok & real).long().cumprod(1).sum(1)
        last = best.gather(1, taken[:, None])[:, 0]
    else:
        x = logits.double() / temp
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
        u = s["uniforms"].double()
        minus = torch.zeros(n, v, dtype=torch.float64, device="cuda")
        taken = torch.zeros_like(counts)
        if t > 1:
            if "draft_logits" in s:
                x = s["draft_logits"].double() / temp
                q = torch.exp(x - x.amax(-1, keepdim=True))
                q /= q.sum(-1, keepdim=True)
            else:
                q = torch.zeros(n, t - 1, v, dtype=torch.float64, device="cuda")
                q.scatter_(2, s["drafts"].long()[:, :, None], 1.0)
            pick = s["drafts"].long()[:, :, None]
            ok = u[:, :-1] * q.gather(2, pick)[:, :, 0] < p[:, :-1].gather(2, pick)[:, :, 0]
            taken = (ok & real).long().cumprod(1).sum(1)
            refused = taken < counts - 1
            of = q.gather(1, taken.clamp_max(t - 2)[:, None, None].expand(n, 1, v))[:, 0]
            minus = torch.where(refused[:, None], of, minus)
        at = taken.clamp_max(t - 1)
        rest = (p.gather(1, at[:, None, None].expand(n, 1, v))[:, 0] - minus).clamp_min(0)
        cum = rest.cumsum(-1)
        last = (cum <= u[:, -1:] * cum[:, -1:]).sum(-1).clamp_max(v - 1)
    ids = torch.full((n, t), -1, dtype=torch.int64, device="cuda")
    if t > 1:
        ids[:, :-1] = torch.where(j[:-1] < taken[:, None], s["drafts"].long(), ids[:, :-1])
    ids.scatter_(1, taken[:, None], last[:, None])
    live = counts > 0
    s["accepted"].copy_(torch.where(live, taken, s["accepted"].long()))
    s["ids"].copy_(torch.where(live[:, None], ids, s["ids"].long()))
    return {"accepted": s["accepted"], "tokens": s["ids"]}


# ------------------------------------------------------ the library's calls --

_kept = {}


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
    hq, hkv, d, theta = HEADS[s["heads"]]
    key = (s["heads"], s["page"], s["window"], s["kv"])
    if key not in _kept:
        _kept[key] = tlm.Paged(ctx, hq, hkv, d, max_tokens=1 << 16, page_tokens=s["page"],
                               inv_freq=_inv_freq(d, theta), sliding_window=s["window"],
                               kv_fmt={"f16": tlm.FMT_F16, "f32": tlm.FMT_F32}[s["kv"]])
    return _kept[key]


def _own(s):
    tlm, ctx = _tlm()
    if "dev" not in s:  # the buffers' addresses, and the batch that names them
        s["dev"] = {k: Dev(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if s["op"] != "verify":
            d = s["dev"]
            s["paged"] = _paged(s)
            s["batch"] = s["paged"].batch(d["k"], d["v"], s["k"].shape[0], d["tables"], s["tables"].shape[1],
                                          d["starts"], s["seqs"], s["tokens"], counts=d["counts"])
    d = s["dev"]
    if s["op"] == "append":
        s["paged"].append(s["batch"], d["x"], d["y"])
        return {"q": s["y"], "k": s["k"], "v": s["v"]}
    if s["op"] == "attention":
        s["paged"].attention(s["batch"], d["x"], d["y"], {"f16": tlm.FMT_F16, "f32": tlm.FMT_F32}[s["out"]])
        return s["y"]
    tlm.verify_drafts(ctx, d["logits"], s["seqs"], s["tokens"], s["vocab"], d["accepted"], d["ids"],
                      drafts=d.get("drafts"), draft_logits=d.get("draft_logits"), counts=d["counts"],
                      uniforms=d["uniforms"], temperature=s["temperature"])
    return {"accepted": s["accepted"], "tokens": s["ids"]}


def run(s):
    if own:
        return _own(s)
    if s["op"] == "append":
        return _append(s)
    if s["op"] == "attention":
        return _attention(s)
    return _verify(s)


# ------------------------------------------------------------------- figures --

def work(case):
    n, t = case["seqs"], case["tokens"]
    if case["op"] == "verify":
        # every row's maximum and sum; the drafts' distributions where there are any
        rows = n - case["idle"]
        values = rows * t * case["vocab"]
        if case["by"] == "model" and case["temperature"] > 0:
            values += rows * (t - 1) * case["vocab"]
        return {"bytes": 4 * values + 16 * rows * t, "flops": 4.0 * values}
    hq, hkv, d, _ = HEADS[case["heads"]]
    starts, counts = _plan(case)
    live = [(s, c) for s, c in zip(starts, counts) if s >= 0]
    rows, size = sum(c for _, c in live), SIZE[case["kv"]]
    if case["op"] == "append":
        return {"bytes": rows * d * ((hq + 2 * hkv) * 4 + 2 * hkv * size + hq * 4), "flops": 6.0 * rows * (hq + hkv) * d}
    keys = sum(s + c - _first(case, s) for s, c in live)
    seen = sum(p + 1 - _first(case, p) for s, c in live for p in range(s, s + c))
    return {"bytes": keys * 2 * hkv * d * size + rows * hq * d * (4 + SIZE[case["out"]]), "flops": 4.0 * hq * d * seen}


# ------------------------------------------------------------------- 64 bits --

def _k_place(tok, dim, page, d, size):
    """Where element (token of the page, dim) of K lies in a page's head."""
    e = 16 // size
    return ((tok // 16) * (d // e) + dim // e) * 16 * e + (tok % 16) * e + dim % e


def _v_place(tok, dim, page, d, size):
    e = 16 // size
    g = 4 * e
    return ((tok // g) * (d // 16) + dim // 16) * 64 * e + ((tok % 16) // 4 * 16 + dim % 16) * e + (tok % g) // 16 * 4 + tok % 4


def _places(case, x, s, first, end, where):
    """Flat indexes [position][kv head][dim] into a pool, of positions first .. end - 1 of sequence s."""
    hq, hkv, d, _ = HEADS[case["heads"]]
    page = case["page"]
    pos = torch.arange(first, end, device="cuda")
    base = x["tables"][s].long()[pos // page] * (hkv * page * d)
    head = torch.arange(hkv, device="cuda") * (page * d)
    dim = torch.arange(d, device="cuda")
    return (base[:, None, None] + head[None, :, None]
            + where((pos % page)[:, None, None], dim[None, None, :], page, d, SIZE[case["kv"]]))


def _exact_append(case, seed):
    hq, hkv, d, theta = HEADS[case["heads"]]
    n, t = case["seqs"], case["tokens"]
    x = _inputs(case, seed)
    starts, counts = _plan(case)
    k, v = x["k"].double(), x["v"].double()
    q = torch.zeros(n, t, hq * d, dtype=torch.float64, device="cuda")
    inv = torch.from_numpy(_inv_freq(d, theta)).cuda().double()
    rows = x["x"].view(n, t, hq + 2 * hkv, d)
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
        k.view(-1)[_places(case, x, s, p0, p0 + c, _k_place)] = z[:, hq:]
        v.view(-1)[_places(case, x, s, p0, p0 + c, _v_place)] = r[:, hq + hkv:]
    return {"q": q, "k": k, "v": v}


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
        k = x["k"].view(-1)[_places(case, x, s, first, p0 + c, _k_place)].double()
        v = x["v"].view(-1)[_places(case, x, s, first, p0 + c, _v_place)].double()
        for j in range(c):
            a, b = _first(case, p0 + j) - first, p0 + j + 1 - first
            kk, vv = k[a:b].repeat_interleave(g, 1), v[a:b].repeat_interleave(g, 1)
            w = torch.softmax((kk * rows[s, j]).sum(-1) / math.sqrt(d), 0)
            y[s, j] = (w[:, :, None] * vv).sum(0).reshape(-1)
    return y


def _exact_verify(case, seed):
    n, t, temp = case["seqs"], case["tokens"], case["temperature"]
    x = _verify_inputs(case, seed)
    accepted, ids = np.zeros(n, np.int32), np.zeros((n, t), np.int32)
    u = x["uniforms"].cpu().numpy().astype(np.float64)
    logits = x["logits"].view(n, t, -1)
    for s, c in enumerate(x["counts"].tolist()):
        if c == 0:
            continue
        ids[s] = -1
        done = False
        for j in range(c):
            row = logits[s, j].double().cpu().numpy()
            tok = int(x["drafts"][s, j]) if j + 1 < c else -1
            if temp == 0:
                best = int(row.argmax())
                ids[s, j] = best
                done = best != tok
            else:
                p = np.exp((row - row.max()) / temp)
                p /= p.sum()
                q = np.zeros_like(p)
                if tok >= 0 and "draft_logits" in x:
                    z = x["draft_logits"][s, j].double().cpu().numpy()
                    q = np.exp((z - z.max()) / temp)
                    q /= q.sum()
                elif tok >= 0:
                    q[tok] = 1
                done = tok < 0 or not u[s, j] * q[tok] < p[tok]
                if done:
                    w = np.maximum(p - q, 0).cumsum()
                    tok = min(int(np.searchsorted(w, u[s, t - 1] * w[-1], side="right")), len(w) - 1)
                ids[s, j] = tok
            if done:
                break
            accepted[s] += 1
    return {"accepted": torch.from_numpy(accepted), "tokens": torch.from_numpy(ids)}


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    return _exact_verify(case, seed)
