"""The paged operators and the verification of drafts together, as a server uses them:
prompts of several chats into pages, steps of one token and its drafts for all chats at
once, a chat that ends and hands its pages to the next.  And the paged calls against
the one-sequence attention op over the same rows."""
import numpy as np
import pytest

import paged_oracle as po
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu

HQ, HKV, D, H, V, PAGE = 8, 2, 64, 256, 480, 32


@pytest.fixture(scope="module")
def ctx():
    c = tlm.Context(0)
    yield c
    c.close()


class Model:
    """One attention layer between an embedding and a head, fp16 weights."""

    def __init__(self, ctx):
        rng = np.random.default_rng(3)
        w = lambda *s: (rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float16)  # noqa: E731
        self.wqkv, self.wo, self.head = w((HQ + 2 * HKV) * D, H), w(H, HQ * D), w(V, H)
        self.emb = rng.standard_normal((V, H)).astype(np.float16)
        self.inv = (1e4 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
        self.lin = [tlm.Linear(ctx, tlm.FMT_F16, m.view(np.uint16)) for m in (self.wqkv, self.wo, self.head)]

    def logits64(self, ids):
        """Logits after every position of `ids`, in 64 bits."""
        x = self.emb[ids].astype(np.float64)
        n = len(ids)
        qkv = (x @ self.wqkv.T.astype(np.float64)).reshape(n, HQ + 2 * HKV, D)
        rot = po.rope(qkv[:, :HQ + HKV], np.arange(n), self.inv)
        out = np.stack([po.attend(rot[p, :HQ], rot[:, HQ:], qkv[:, HQ + HKV:], p, 0, D ** -0.5) for p in range(n)])
        return (x + out.reshape(n, -1) @ self.wo.T.astype(np.float64)) @ self.head.T.astype(np.float64)


class Server:
    """Pages, tables and lengths of some chats; step() computes rows for all of them."""

    def __init__(self, ctx, model, slots, pages, width):
        self.ctx, self.m, self.slots, self.width, self.pages = ctx, model, slots, width, pages
        self.paged = tlm.Paged(ctx, HQ, HKV, D, width * PAGE, page_tokens=PAGE, inv_freq=model.inv)
        n = pages * self.paged.page_bytes()
        self.kp = ctx.array(np.full(n // 2, np.nan, np.float16))  # no page holds anything yet
        self.vp = ctx.array(np.full(n // 2, np.nan, np.float16))
        self.free = list(np.random.default_rng(1).permutation(pages))
        self.tables = np.full((slots, width), -1, np.int32)
        self.length = np.full(slots, -1, np.int32)  # tokens in the cache; -1: idle

    def end(self, s):
        self.free += [p for p in self.tables[s] if p >= 0]
        self.tables[s], self.length[s] = -1, -1

    def step(self, ids, counts):
        """ids [slots][t], counts per slot (0: nothing): logits buffer of all rows."""
        t = ids.shape[1]
        for s in range(self.slots):
            for p in range(-(-(max(self.length[s], 0) + counts[s]) // PAGE)):
                if counts[s] and self.tables[s, p] < 0:
                    self.tables[s, p] = self.free.pop()
        c, rows = self.ctx, self.slots * t
        x = self.m.emb[ids.reshape(-1)]
        qkv, q = c.buffer(4 * rows * (HQ + 2 * HKV) * D), c.buffer(4 * rows * HQ * D)
        att = c.array(np.zeros((rows, HQ * D), np.float16))
        y = c.buffer(4 * rows * H)
        self.counts = c.array(np.asarray(counts, np.int32))
        b = self.paged.batch(self.kp, self.vp, self.pages, c.array(self.tables), self.width, c.array(self.length),
                             self.slots, t, self.counts)
        self.m.lin[0].rows(c.array(x.view(np.uint16)), rows, qkv)
        self.paged.append(b, qkv, q)
        self.paged.attention(b, q, att)
        self.m.lin[1].rows(att, rows, y)
        hidden = (x.astype(np.float32) + y.read().reshape(rows, H)).astype(np.float16)
        logits = c.buffer(4 * rows * V)
        self.m.lin[2].rows(c.array(hidden.view(np.uint16)), rows, logits)
        return logits

    def verify(self, logits, ids, counts, temperature, uniforms=None):
        t, c = ids.shape[1], self.ctx
        acc, out = c.array(np.full(self.slots, -9, np.int32)), c.array(np.full((self.slots, t), -9, np.int32))
        tlm.verify_drafts(c, logits, self.slots, t, V, acc, out, counts=self.counts, temperature=temperature,
                          drafts=c.array(np.ascontiguousarray(ids[:, 1:])) if t > 1 else None,
                          uniforms=None if uniforms is None else c.array(uniforms))
        return acc.read(np.int32), out.read(np.int32).reshape(self.slots, t)


# Rounded to fp16 on the way to the logits: K, V, the attention's output and the hidden
# row, each by 2^-11 of its size; 256 products with the head's weights of 1/16 add up
# to about 10 in magnitudes, and the layer passes its share on at about the same size:
# 8 roundings of 10 * 2^-11 at the very worst.
TOL = 8 * 10 * 2.0 ** -11


def emitted_are_greedy(model, ids, start):
    """Every token from `start` on is the 64-bit model's best after those before it, but for roundings."""
    ref = model.logits64(ids)
    for p in range(start, len(ids)):
        row = ref[p - 1]
        assert row[ids[p]] >= row.max() - TOL, f"token {p}: {row.max() - row[ids[p]]}"


def test_speculative_greedy_decoding_of_several_chats(ctx):
    model = Model(ctx)
    rng = np.random.default_rng(8)
    prompts = [list(rng.integers(0, V, n)) for n in (45, 3, 64, 1)]
    slots, width, total = 4, 5, 100
    sv = Server(ctx, model, slots, 24, width)
    # the prompts at once, padded to the longest; the last slot comes later
    first = [prompts[0], prompts[1], prompts[2], []]
    t = max(len(p) for p in first)
    ids = np.zeros((slots, t), np.int64)
    for s, p in enumerate(first):
        ids[s, :len(p)] = p
    counts = np.array([len(p) for p in first])
    sv.length = np.array([0, 0, 0, -1], np.int32)
    logits = sv.step(ids, counts).read().reshape(slots, t, V)
    chats = [list(p) for p in first]
    for s in range(3):
        chats[s].append(int(logits[s, counts[s] - 1].argmax()))
        sv.length[s] = counts[s]
    joined = False
    taken_all = refused_all = 0
    for step in range(60):
        if step == 6:  # the short chat ends, another one starts in the idle slot, on its pages
            done = chats[1]
            sv.end(1)
            chats[1] = None
            chats[3] = list(prompts[3])
            sv.length[3] = 0
            joined = True
        live = [s for s in range(slots) if chats[s] and len(chats[s]) < total]
        if not live:
            break
        k = int(rng.integers(1, 5))
        ids, counts = np.zeros((slots, k), np.int64), np.zeros(slots, np.int64)
        for s in live:
            counts[s] = min(int(rng.integers(1, k + 1)), total - len(chats[s]))
            ids[s, 0] = chats[s][-1]
            if counts[s] > 1:  # drafts: what the 64-bit model goes on with, now and then something else
                ctx_ids = list(chats[s])
                for j in range(1, counts[s]):
                    ctx_ids.append(int(model.logits64(ctx_ids)[-1].argmax()) if rng.random() < 0.7 else int(rng.integers(V)))
                    ids[s, j] = ctx_ids[-1]
        start = sv.length.copy()
        start[[s for s in range(slots) if s not in live]] = -1
        keep, sv.length = sv.length, start
        logits = sv.step(ids, counts)
        acc, out = sv.verify(logits, ids.astype(np.int32), counts, 0.0)
        sv.length = keep
        for s in range(slots):
            if s not in live:
                assert acc[s] == -9 and np.all(out[s] == -9)
                continue
            assert 0 <= acc[s] < counts[s]
            taken_all += acc[s]
            refused_all += acc[s] < counts[s] - 1
            chats[s] += [int(x) for x in out[s, :acc[s] + 1]]
            sv.length[s] += acc[s] + 1
            assert np.all(out[s, acc[s] + 1:] == -1)
    sv.paged.status()
    assert joined and taken_all > 10 and refused_all > 5
    for ids, p in ((chats[0], prompts[0]), (done, prompts[1]), (chats[2], prompts[2]), (chats[3], prompts[3])):
        assert len(ids) > len(p) + 5
        emitted_are_greedy(model, ids, len(p))
    sv.paged.close()


def test_sampled_tokens_are_those_of_the_given_numbers(ctx):
    """Sampling with drafts: what is emitted follows from the logits and the random numbers that were given."""
    model = Model(ctx)
    rng = np.random.default_rng(9)
    sv = Server(ctx, model, 3, 12, 3)
    sv.length = np.zeros(3, np.int32)
    for step in range(12):
        t = 4
        ids, counts = rng.integers(0, V, (3, t)), np.array([4, 1 + step % 4, 2])
        u = rng.random((3, t), np.float32)
        logits = sv.step(ids, counts)
        acc, out = sv.verify(logits, ids.astype(np.int32), counts, 0.7, u)
        ra, ro = po.verify(logits.read().reshape(3, t, V), ids[:, 1:], counts, u, 0.7)
        assert np.array_equal(acc, ra) and np.array_equal(out, ro)
        sv.length += acc + 1
    sv.paged.status()
    sv.paged.close()


@pytest.mark.parametrize("hq,hkv,d,window", [(14, 2, 64, 0), (24, 8, 128, 0), (8, 2, 64, 100)])
def test_the_same_rows_through_the_one_sequence_op(ctx, hq, hkv, d, window):
    """A prompt and the tokens after it, paged and in an Attention's own cache: the V rows are the same to the bit (one
    rounding of the same value), the decoded outputs agree to 32 bits, the prompt's to the batched op's fp16 queries
    and probabilities (2^-10 of scores of order ten).  A K element is a c + b s of 32-bit values, and which of the
    products is rounded before the sum is each kernel's own: two results differ by at most 2 * 2^-24 (|a| + |b|), and
    each is then rounded by at most 2^-11 of itself (2^-25 below fp16's normal range): 2^-10 |k| + 2^-24 and that
    difference, |a| and |b| at most the largest input."""
    n, page = 333, 64
    rng = np.random.default_rng(hq)
    inv = (1e4 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    x = rng.standard_normal((n + 5, (hq + 2 * hkv) * d)).astype(np.float32)
    one = tlm.Attention(ctx, hq, hkv, d, n + 5, inv_freq=inv, sliding_window=window)
    paged = tlm.Paged(ctx, hq, hkv, d, 512, page_tokens=page, inv_freq=inv, sliding_window=window)
    pages = 8
    kp, vp = (ctx.array(np.zeros(pages * hkv * page * d, np.float16)) for _ in range(2))
    table = rng.permutation(pages).astype(np.int32)
    q, out = ctx.buffer(4 * n * hq * d), ctx.buffer(4 * n * hq * d)
    ref = ctx.buffer(2 * n * hq * d)

    def batch(start, rows):
        return paged.batch(kp, vp, pages, ctx.array(table), pages, ctx.array(np.array([start], np.int32)), 1, rows)

    b = batch(0, n)
    paged.append(b, ctx.array(x[:n]), q)
    paged.attention(b, q, out)
    got = out.read(np.float16)[:n * hq * d].astype(np.float32)
    one.rows(ctx.array(x[:n]), n, 0, ref)
    want = ref.read(np.float16).astype(np.float32)
    assert np.abs(got - want).max() <= 2.0 ** -10 * 10 * np.abs(x).max()
    y = ctx.buffer(4 * hq * d)
    for p in range(n, n + 5):
        b = batch(p, 1)
        paged.append(b, ctx.array(x[p]), q)
        paged.attention(b, q, out, tlm.FMT_F32)
        got = out.read()[:hq * d]
        want = one(ctx.array(x[p]), p, y).read()
        assert np.abs(got - want).max() <= 2e-5 * max(1.0, np.abs(want).max())
    paged.status()
    k, v = one.read_cache(n + 5)
    at = po.places(table, np.arange(n + 5), hkv, page, d, 8, po.k_at)
    got = kp.read(np.float16)[at].reshape(n + 5, -1).astype(np.float64)
    assert np.all(np.abs(got - k) <= 2.0 ** -10 * np.maximum(np.abs(got), np.abs(k)) + 2.0 ** -24
                  + 2 * 2.0 ** -24 * 2 * np.abs(x).max())
    at = po.places(table, np.arange(n + 5), hkv, page, d, 8, po.v_at)
    assert np.array_equal(vp.read(np.float16)[at].reshape(n + 5, -1).astype(np.float32), v)
    one.close()
    paged.close()
