"""Paged append and attention against 64-bit forms (paged_oracle.py), at the sizes and
tables where they can go wrong.  The pool holds NaN wherever no sequence's position
lies, tables hold -1 wherever no page is needed.

Tolerances.  Append: the angles' cos and sin are rounded to 32 bits and the products
and their sum round three times: 4 * 2^-24 of |a| + |b|, then half a step of the
cache's type.  Attention: a score is a 32-bit sum of d products over at most d / 4
steps, q exact to 2^-22 of its row's largest element: off by (d / 4 + 8) 2^-24 A, A the
largest sum of |q k| scale; the output, a mean of v under weights each off by twice
that, and a 32-bit sum in steps of 16 or more positions over at most 16 waves and 64
chunks: (2 (d / 4 + 8) A + n / 16 + 96) 2^-24 max |v|, then half a step of its type."""
import ctypes

import numpy as np
import pytest

import paged_oracle as po
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HALF = {tlm.FMT_F16: 2.0 ** -11, tlm.FMT_F32: 2.0 ** -24}
NP = {tlm.FMT_F16: np.float16, tlm.FMT_F32: np.float32}


@pytest.fixture(scope="module")
def ctx():
    c = tlm.Context(0)
    yield c
    c.close()


class Serving:
    """Sequences with caches of random rows, on the host and in a pool on the device."""

    def __init__(self, ctx, hq, hkv, d, lengths, tokens, page=32, kv=tlm.FMT_F16, window=0, counts=None, seed=0,
                 rotary=None, spare=2, factor=1.0, scale=0.0, max_tokens=None):
        self.ctx, self.hq, self.hkv, self.d, self.page, self.kv, self.window = ctx, hq, hkv, d, page, kv, window
        rng = self.rng = np.random.default_rng([seed, hq, d, page, tokens])
        self.n, self.tokens, self.starts = len(lengths), tokens, np.array(lengths, np.int32)
        self.counts = None if counts is None else np.array(counts, np.int32)
        self.rows = [0 if s < 0 else tokens if counts is None else min(max(counts[i], 0), tokens)
                     for i, s in enumerate(lengths)]
        ends = [max(s, 0) + r if r else 0 for s, r in zip(lengths, self.rows)]
        firsts = [max(0, s - window + 1) // page if window else 0 for s in lengths]
        self.width = max(1, max(-(-e // page) for e in ends))
        need = sum(max(0, -(-e // page) - f) for e, f in zip(ends, firsts))
        self.pages = need + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((self.n, self.width), -1, np.int32)
        at = 0
        for s, (e, f) in enumerate(zip(ends, firsts)):
            m = max(0, -(-e // page) - f)
            if m:
                self.tables[s, f:f + m] = order[at:at + m]
                at += m
        rd = d if rotary is None else rotary
        self.inv = (1e4 ** (-np.arange(0, rd, 2) / rd)).astype(np.float32) if rd else None
        self.factor, self.scale = factor, scale or d ** -0.5
        self.paged = tlm.Paged(ctx, hq, hkv, d, max_tokens or self.width * page, page_tokens=page, inv_freq=self.inv,
                               rotary_dim=rd or None, sliding_window=window, kv_fmt=kv, attention_factor=factor,
                               attn_scale=scale)
        self.e = 4 if kv == tlm.FMT_F32 else 8
        t = NP[kv]
        self.k = [rng.standard_normal((e, hkv, d)).astype(t) for e in ends]
        self.v = [rng.standard_normal((e, hkv, d)).astype(t) for e in ends]
        self.firsts = [f * page for f in firsts]

    def pools(self, upto):
        """Host pools with positions [first page, upto[s]) of every sequence, NaN elsewhere."""
        kp = np.full(self.pages * self.hkv * self.page * self.d, np.nan, NP[self.kv])
        vp = kp.copy()
        for s in range(self.n):
            pos = np.arange(self.firsts[s], max(upto[s], self.firsts[s]) if self.rows[s] else self.firsts[s])
            if pos.size:
                kp[po.places(self.tables[s], pos, self.hkv, self.page, self.d, self.e, po.k_at)] = self.k[s][pos]
                vp[po.places(self.tables[s], pos, self.hkv, self.page, self.d, self.e, po.v_at)] = self.v[s][pos]
        return kp, vp

    def upload(self, kp, vp):
        self.kb, self.vb = self.ctx.array(kp), self.ctx.array(vp)
        self.batch = self.paged.batch(self.kb, self.vb, self.pages, self.ctx.array(self.tables), self.width,
                                      self.ctx.array(self.starts), self.n, self.tokens,
                                      None if self.counts is None else self.ctx.array(self.counts))
        return self.batch

    def attention(self, q, out_fmt):
        out = self.ctx.array(np.full((self.n, self.tokens, self.hq * self.d), 77, NP[out_fmt]))
        self.paged.attention(self.batch, self.ctx.array(q), out, out_fmt)
        return out.read(NP[out_fmt]).reshape(self.n, self.tokens, self.hq, self.d)

    def check(self, q, got, out_fmt, there=None, reported=False):
        if not reported:
            self.paged.status()
        for s in range(self.n):
            assert np.all(got[s, self.rows[s]:] == 77), f"rows behind sequence {s}"
            for j in range(self.rows[s]):
                pos = int(self.starts[s]) + j
                first = max(0, pos - self.window + 1) if self.window else 0
                ref = po.attend(q[s, j], self.k[s], self.v[s], pos, self.window, self.scale,
                                None if there is None else there[s])
                kk = np.abs(self.k[s][first:pos + 1].astype(np.float64)).repeat(self.hq // self.hkv, 1)
                big = max(1.0, float((kk * np.abs(q[s, j])).sum(-1).max()) * self.scale)
                mv = float(np.abs(self.v[s][first:pos + 1].astype(np.float64)).max())
                tol = (2 * (self.d / 4 + 8) * big + (pos - first + 1) / 16 + 96) * EPS * mv + HALF[out_fmt] * np.abs(ref)
                err = np.abs(got[s, j].astype(np.float64) - ref)
                assert np.all(err <= tol + 2.0 ** -25), f"sequence {s} row {j}: {np.nanmax(err - tol)} over {err.max()}"

    def close(self):
        self.paged.close()


def normal(sv):
    return sv.rng.standard_normal((sv.n, sv.tokens, sv.hq, sv.d)).astype(np.float32)


def attend(sv, out_fmt=tlm.FMT_F32):
    sv.upload(*sv.pools([s + r if r else 0 for s, r in zip(sv.starts, sv.rows)]))
    q = normal(sv)
    got = sv.attention(q, out_fmt)
    more = sv.counts is not None and bool(np.any((sv.counts > sv.tokens) & (sv.starts >= 0)))
    if more:  # a count above the batch's rows is reported, the rows that there are computed
        with pytest.raises(tlm.TlmError) as e:
            sv.paged.status()
        assert e.value.code == tlm.TLM_ERR_RANGE
    sv.check(q, got, out_fmt, reported=more)
    sv.close()


# ------------------------------------------------------------------- append --

def append(sv, want_q=True):
    kp, vp = sv.pools(np.maximum(sv.starts, 0))
    sv.upload(kp, vp)
    x = sv.rng.standard_normal((sv.n, sv.tokens, sv.hq + 2 * sv.hkv, sv.d)).astype(np.float32)
    q = sv.ctx.array(np.full((sv.n, sv.tokens, sv.hq, sv.d), 77, np.float32))
    sv.paged.append(sv.batch, sv.ctx.array(x), q if want_q else None)
    got_q = q.read().reshape(sv.n, sv.tokens, sv.hq, sv.d)
    got_k, got_v = sv.kb.read(NP[sv.kv]), sv.vb.read(NP[sv.kv])
    sv.paged.status()
    touched = np.zeros(kp.size, bool), np.zeros(kp.size, bool)
    half = HALF[sv.kv]
    tiny = 2.0 ** -25 if sv.kv == tlm.FMT_F16 else 0.0  # half the smallest step of fp16
    for s in range(sv.n):
        r = sv.rows[s]
        if want_q:
            assert np.all(got_q[s, r:] == 77)
        else:
            assert np.all(got_q == 77)
        if not r:
            continue
        pos = int(sv.starts[s]) + np.arange(r)
        rot = po.rope(x[s, :r, :sv.hq + sv.hkv], pos, sv.inv, sv.factor)
        h = 0 if sv.inv is None else sv.inv.size
        mag = np.abs(x[s, :r, :sv.hq + sv.hkv]).astype(np.float64)
        mag[..., :2 * h] = np.concatenate([mag[..., :h] + mag[..., h:2 * h]] * 2, -1) * max(1.0, sv.factor)
        tol = 4 * EPS * mag
        if want_q:
            assert np.all(np.abs(got_q[s, :r] - rot[:, :sv.hq]) <= tol[:, :sv.hq]), f"q of sequence {s}"
        at = po.places(sv.tables[s], pos, sv.hkv, sv.page, sv.d, sv.e, po.k_at)
        kk = got_k[at].astype(np.float64)
        assert np.all(np.abs(kk - rot[:, sv.hq:]) <= tol[:, sv.hq:] + half * np.abs(rot[:, sv.hq:]) * 1.001 + tiny), f"k of {s}"
        touched[0][at] = True
        at = po.places(sv.tables[s], pos, sv.hkv, sv.page, sv.d, sv.e, po.v_at)
        assert np.array_equal(got_v[at], x[s, :r, sv.hq + sv.hkv:].astype(NP[sv.kv])), f"v of {s}"
        touched[1][at] = True
    for got, was, t in ((got_k, kp, touched[0]), (got_v, vp, touched[1])):
        assert np.array_equal(got[~t], was[~t], equal_nan=True), "elements of no new position"
    sv.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(14, 2, 64, 64), (24, 8, 128, 32), (4, 4, 32, 128), (6, 1, 96, 32)])
@pytest.mark.parametrize("tokens", [1, 5, 45])
def test_append(ctx, hq, hkv, d, page, kv, tokens):
    counts = [tokens, 1, max(1, tokens - 3), 0, tokens]
    append(Serving(ctx, hq, hkv, d, [0, 63, 30, 12, -1], tokens, page, kv, counts=counts))


@pytest.mark.parametrize("tokens", [31, 32, 33, 64, 100, 300])
@pytest.mark.parametrize("start", [0, 1, 16, 31, 45])
def test_append_chunks_at_group_edges(ctx, tokens, start):
    append(Serving(ctx, 4, 2, 64, [start, start + 7], tokens, 32, tlm.FMT_F16, counts=[tokens, tokens - 2]))


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("rotary", [0, 2, 20, 32, 48])
@pytest.mark.parametrize("tokens", [1, 70])
def test_append_partial_rotary_and_no_q(ctx, kv, rotary, tokens):
    append(Serving(ctx, 3, 1, 64, [9, 40], tokens, 64, kv, rotary=rotary, factor=1.25))
    append(Serving(ctx, 3, 1, 64, [9, 40], tokens, 64, kv, rotary=rotary), want_q=False)


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_append_far_positions(ctx, kv):
    """Angles of positions past 2^16, each row the last of a page or the first of one."""
    append(Serving(ctx, 2, 1, 128, [100000, 99999, 65535, 131071], 2, 128, kv, window=40, max_tokens=1 << 18))


# ---------------------------------------------------------------- attention --

@pytest.mark.parametrize("out_fmt", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(14, 2, 64, 64), (24, 8, 128, 32), (4, 4, 32, 128), (16, 1, 96, 32)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_attention_shapes(ctx, hq, hkv, d, page, kv, out_fmt, tokens):
    attend(Serving(ctx, hq, hkv, d, [0, 15, 31, 32, 200, -1, 517], tokens, page, kv,
                   counts=[tokens, tokens, 1, tokens, 2, 1, tokens]), out_fmt)


@pytest.mark.parametrize("start", [0, 1, 14, 15, 16, 30, 31, 32, 33, 63, 64, 127, 255, 256, 257, 511, 512, 1000, 2047, 2048])
@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_attention_lengths(ctx, start, kv):
    attend(Serving(ctx, 8, 2, 64, [start], 1, 64, kv))


@pytest.mark.parametrize("tokens", [2, 4, 5, 7, 16, 17, 40, 130])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (24, 8, 128), (14, 2, 64), (16, 1, 128)])
def test_attention_drafts_and_chunks(ctx, tokens, hq, hkv, d):
    attend(Serving(ctx, hq, hkv, d, [0, 29, 300], tokens, 32, tlm.FMT_F16, counts=[tokens, tokens, max(1, tokens - 1)]))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 600])
@pytest.mark.parametrize("tokens", [1, 6])
@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_attention_windows(ctx, window, tokens, kv):
    """The pages before a window are given back: -1 in the tables, NaN in the pool."""
    attend(Serving(ctx, 8, 2, 64, [0, window - 1, window, window + 45, 1500], tokens, 32, kv, window=window))


@pytest.mark.parametrize("n", [65, 130, 300])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (8, 8)])
def test_attention_long_caches_among_many(ctx, n, hq, hkv):
    """Some sequences in several chunks, in every group of 64 that a block looks through."""
    rng = np.random.default_rng(n + hq)
    lengths = [int(x) for x in rng.integers(0, 60, n)]
    for s in (1, 63, 64, n - 2, n - 1):
        lengths[s] = 3000 + 7 * s
    lengths[5] = -1
    attend(Serving(ctx, hq, hkv, 64, lengths, 1, 64))


@pytest.mark.parametrize("n", [1, 63, 64, 65, 200])
def test_attention_many_sequences_of_all_lengths(ctx, n):
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in np.exp(rng.uniform(0, np.log(900), n))]
    for s in range(0, n, 7):
        lengths[s] = -1 if s else lengths[s]
    attend(Serving(ctx, 4, 2, 64, lengths, 1, 32))


@pytest.mark.parametrize("n,hq,hkv,tokens", [(384, 8, 8, 1), (385, 4, 2, 1), (1024, 2, 1, 1), (1500, 4, 4, 2), (4500, 2, 1, 1)])
@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_attention_of_more_sequences_than_a_wave_plans(ctx, n, hq, hkv, tokens, kv):
    """Long caches in several chunks among many short ones and idle slots, whole groups of 64 of them; a row past the
    model's positions is reported."""
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in rng.integers(0, 40, n)]
    for s in (1, 63, 64, n // 2, n - 70, n - 1):
        lengths[s] = 2500 + 5 * (s % 64)
    for s in range(128, 256):
        lengths[s] = -1
    attend(Serving(ctx, hq, hkv, 32, lengths, tokens, 32, kv, counts=[int(x) for x in rng.integers(0, tokens + 1, n)]))
    sv = Serving(ctx, hq, hkv, 32, [3] * n, 1, 32, kv, max_tokens=40)
    sv.upload(*sv.pools(sv.starts + 1))
    starts = sv.starts.copy()
    starts[n - 3] = 40
    sv.batch.starts = ctx.array(starts).ptr
    sv.rows[n - 3] = 0
    q = normal(sv)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, reported=True)
    with pytest.raises(tlm.TlmError) as e:
        sv.paged.status()
    assert e.value.code == tlm.TLM_ERR_RANGE and "left out" in str(e.value)
    sv.close()


def test_attention_of_2_22_sequences(ctx):
    """The most sequences that a call takes, over tables that name two pages: K is 0 and V 0 in one page and 1 in the
    other, so an output is the share of a sequence's positions in the second.  32-bit sums of up to 1500 ones are exact,
    one division is not."""
    n, page, d, width = 1 << 22, 512, 32, 3
    rng = np.random.default_rng(0)
    paged = tlm.Paged(ctx, 1, 1, d, width * page, page_tokens=page)
    k, v = np.zeros(2 * page * d, np.float16), np.repeat([0, 1], page * d).astype(np.float16)
    tables = rng.integers(0, 2, (n, width)).astype(np.int32)
    starts = rng.integers(-1, 20, n).astype(np.int32)
    long = rng.integers(0, n, 300)
    starts[long] = rng.integers(0, 1500, 300)
    starts[n - 1] = 1400
    q, out = ctx.buffer(4 * n * d), ctx.buffer(2 * n * d)
    q.write(np.ones((n, d), np.float32))
    out.write(np.full((n, d), 77, np.float16))
    batch = paged.batch(ctx.array(k), ctx.array(v), 2, ctx.array(tables), width, ctx.array(starts), n)
    paged.attention(batch, q, out)
    paged.status()
    got = out.read(np.float16).reshape(n, d)
    seen = np.clip((starts + 1)[:, None] - page * np.arange(width), 0, page)
    ref = (seen * tables).sum(1) / np.maximum(starts + 1, 1)
    ref = np.where(starts < 0, 77, ref)
    assert np.all(np.abs(got - ref[:, None]) <= ref[:, None] * (2.0 ** -11 + 2.0 ** -22))
    q.free()
    out.free()
    paged.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("tokens", [1, 5])
def test_attention_one_long_cache_among_short_ones(ctx, kv, tokens):
    attend(Serving(ctx, 8, 2, 128, [20000, 3, 700], tokens, 256, kv))


def test_attention_of_few_rows_in_a_batch_with_room_for_many(ctx):
    """Room for 8192 rows and 40 of them there: so many row groups leave no room for partial results, and a sequence is
    one block's however long it is."""
    attend(Serving(ctx, 16, 16, 32, [1500, 2, -1], 8192, 64, counts=[40, 3, 5]))


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_attention_over_2_30_positions(ctx, kv):
    """40 sequences of up to 2^30 positions (their tiles together pass 32 bits), three of them as long as that over
    tables that name the same pages again and again.  K is 0 and V 0 or 1, ones in a 256th of the table: every sum is a
    count.  A sequence's 2^30 is joined from at most 256 chunks of 8 waves, a rounding each, and one division."""
    n, page, d, width, part = 40, 1024, 32, 1 << 20, 1 << 12
    paged = tlm.Paged(ctx, 1, 1, d, 1 << 30, page_tokens=page, kv_fmt=kv)
    k, v = np.zeros(2 * page * d, NP[kv]), np.repeat([0, 1], page * d).astype(NP[kv])
    tables = np.zeros((n, width), np.int32)
    starts = np.array([37 * s if s % 5 else -1 for s in range(n)], np.int32)
    tables[1::2] = 1
    for s, at in ((3, 0), (8, width // 2 + 5 * part + 77), (39, width - part)):
        starts[s] = (1 << 30) - 1 - s
        tables[s] = 0
        tables[s, at:at + part] = 1
    out = ctx.array(np.full((n, d), 77, np.float32))
    batch = paged.batch(ctx.array(k), ctx.array(v), 2, ctx.array(tables), width, ctx.array(starts), n)
    paged.attention(batch, ctx.array(np.ones((n, d), np.float32)), out, tlm.FMT_F32)
    paged.status()
    got = out.read(np.float32).reshape(n, d).astype(np.float64)
    for s in range(n):
        if starts[s] < 0:
            ref = 77.0
        elif starts[s] < 1 << 20:
            ref = float(tables[s, 0])
        else:
            ones = part * page - (s if s == 39 else 0)
            ref = ones / (starts[s] + 1.0)
        assert np.all(np.abs(got[s] - ref) <= 272 * EPS * ref), (s, got[s, 0], ref)


@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** 18, 2.0 ** 60])
@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
def test_queries_of_any_size(ctx, size, kv):
    """q past fp16's range over keys that make scores of order ten, each row of a size of its own."""
    sv = Serving(ctx, 4, 2, 64, [400], 2, 64, kv, scale=1.0)
    if kv == tlm.FMT_F16 and size > 2.0 ** 20:
        sv.k = [(k.astype(np.float64) * 2.0 ** -14).astype(np.float16) for k in sv.k]
        size = 2.0 ** 14
    elif size > 1:
        sv.k = [(k.astype(np.float64) / size).astype(NP[kv]) for k in sv.k]
    sv.upload(*sv.pools(sv.starts + 2))
    q = normal(sv) * np.float32(size)
    q[0, 1, 2] *= np.float32(2.0 ** -30)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32)
    sv.close()


def test_no_spread_and_one_certain_key(ctx):
    """All scores equal (q = 0), and a key whose score passes the rest by hundreds, late and early."""
    sv = Serving(ctx, 4, 2, 64, [700, 700, 700], 1, 64)
    sv.k[1][650] = 30
    sv.k[2][3] = 30
    sv.upload(*sv.pools(sv.starts + 1))
    q = np.abs(normal(sv))
    q[0] = 0
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32)
    sv.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 23, 2.0 ** 26, 2.0 ** 30, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(ctx, size, sign, kv):
    """Scores past what a 32-bit number holds in whole steps, above and below 0: the best key's V, and nothing else.
    The best two keys' scores are at least a 64th of the largest apart, far more than they are off by."""
    sv = Serving(ctx, 4, 2, 64, [300, 40], 3, 64, kv, scale=1.0)
    for k in sv.k:
        k[..., 1:] = 0
        for h in range(2):  # 1 .. 2 in steps of a 512th, each once, and one 2 + a 32nd (or, below 0, 1 - a 64th)
            k[:, h, 0] = 1 + sv.rng.permutation(512)[:k.shape[0]] / 512
            k[sv.rng.integers(0, 38), h, 0] = 2 + 1 / 32 if sign > 0 else 1 - 1 / 64
    sv.upload(*sv.pools(sv.starts + 3))
    q = np.zeros((2, 3, 4, 64), np.float32)
    q[..., 0] = sign * size * (1 + np.arange(4) / 7)
    got = sv.attention(q, tlm.FMT_F32)
    sv.paged.status()
    for s in range(2):
        for h in range(4):
            best = np.argmax(sign * sv.k[s][:38, h // 2, 0])
            want = sv.v[s][best, h // 2].astype(np.float64)
            assert np.all(np.abs(got[s, :, h] - want) <= 2.0 ** -21 * np.abs(want)), (s, h)
    sv.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("tokens", [1, 3])
def test_small_elements_of_q_beside_a_large_one(ctx, kv, tokens):
    """Elements 2^-20 of the row's largest decide the scores: K is 0 where q is large and of 2^13 elsewhere.  An element
    is off by 2^-22 of itself or 2^-39 of the largest (1), so a score by A 2^-22 + 2^-39 sum |k| scale and a 32-bit sum's
    (d / 4 + 8) 2^-24 A; the output as elsewhere."""
    scale = 64.0
    sv = Serving(ctx, 4, 2, 64, [700, 90], tokens, 64, kv, scale=scale)
    for k in sv.k:
        k *= NP[kv](2.0 ** 13)
        k[..., 0] = 0
    sv.upload(*sv.pools(sv.starts + tokens))
    q = normal(sv) * np.float32(2.0 ** -20)
    q[..., 0] = 1
    got = sv.attention(q, tlm.FMT_F32).astype(np.float64)
    sv.paged.status()
    for s in range(2):
        for j in range(tokens):
            n = int(sv.starts[s]) + j + 1
            ref = po.attend(q[s, j], sv.k[s], sv.v[s], n - 1, 0, scale)
            kk = np.abs(sv.k[s][:n].astype(np.float64)).repeat(2, 1)
            a = float((kk * np.abs(q[s, j])).sum(-1).max()) * scale
            off = (4 + 16 + 8) * EPS * a + 2.0 ** -39 * float(kk.sum(-1).max()) * scale
            mv = float(np.abs(sv.v[s][:n].astype(np.float64)).max())
            tol = (2 * off + (n / 16 + 96) * EPS) * mv
            err = np.abs(got[s, j] - ref).max()
            assert err <= tol, f"sequence {s} row {j}: {err} over {tol}"
    sv.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("octaves", [18.4, 22.4, 25.6])
@pytest.mark.parametrize("every", [0, 32])
def test_small_weights_beside_dominant_keys(ctx, kv, octaves, every):
    """One key, or one in 32, weighs 2^octaves times each of the others, and has V = 0: the output is what the small
    weights w bring.  All terms are positive, so errors are relative.  A weight is off by g = octaves ln 2 times q's
    2^-22 and the scale's and score's three roundings, and exp2's 2^-23: 8 g + 2 of 2^-24; as a pair by 2^-22 or
    2^-39 of the largest; numerator and denominator each by n / 16 + 96 roundings."""
    sv = Serving(ctx, 4, 2, 64, [700, 5000], 1, 64, kv, scale=1.0)
    for k, v in zip(sv.k, sv.v):
        k[:] = 0
        v[:] = sv.rng.uniform(0.5, 1, v.shape)
        at = slice(5, None, every) if every else [5]
        k[at, :, 0], v[at] = 1, 0
    sv.upload(*sv.pools(sv.starts + 1))
    gap = octaves * np.log(2)
    q = sv.rng.uniform(0, 1, (2, 1, 4, 64)).astype(np.float32)
    q[..., 0] = gap
    got = sv.attention(q, tlm.FMT_F32).astype(np.float64)
    sv.paged.status()
    for s in range(2):
        n = int(sv.starts[s]) + 1
        ref = po.attend(q[s, 0], sv.k[s], sv.v[s], n - 1, 0, 1.0)
        tol = (8 * gap + 2 + 4 + 2 * (n / 16 + 96)) * EPS + 2.0 ** (octaves - 39)
        assert np.all(np.abs(got[s, 0] - ref) <= tol * ref), (s, np.abs(got[s, 0] / ref - 1).max(), tol)
    sv.close()


@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hq", [2, 16])
def test_masked_rows_of_drafts_are_not_seen(ctx, kv, bad, hq):
    """A draft whose K and V are not finite does not reach the rows before it, nor the rows whose window has passed it."""
    sv = Serving(ctx, hq, 1, 64, [45], 6, 32, kv, window=4)
    sv.k[0][48], sv.v[0][48, :, 5] = bad, bad
    sv.upload(*sv.pools(sv.starts + 6))
    q = normal(sv)
    got = sv.attention(q, tlm.FMT_F32)
    for j in (0, 1, 2):  # positions 45 .. 47
        ref = po.attend(q[0, j], sv.k[0], sv.v[0], 45 + j, 4, sv.scale)
        assert np.abs(got[0, j] - ref).max() <= 1e-4, f"row {j}"
    assert not np.isfinite(got[0, 3:, :, 5]).any()
    sv.close()
    sv = Serving(ctx, hq, 1, 64, [45], 6, 32, kv, window=2)
    sv.v[0][46, :, 7] = bad
    sv.upload(*sv.pools(sv.starts + 6))
    got = sv.attention(q, tlm.FMT_F32)
    for j in (0, 3, 4, 5):
        ref = po.attend(q[0, j], sv.k[0], sv.v[0], 45 + j, 2, sv.scale)
        assert np.abs(got[0, j] - ref).max() <= 1e-4, f"row {j} of the passed window"
    sv.close()


def test_a_query_that_is_not_finite_stays_in_its_row(ctx):
    sv = Serving(ctx, 4, 2, 64, [100], 2, 32)
    sv.upload(*sv.pools(sv.starts + 2))
    q = normal(sv)
    q[0, 0, 1, 3] = np.nan
    got = sv.attention(q, tlm.FMT_F32)
    assert np.isnan(got[0, 0, 1]).all()
    q2, got2 = q.copy(), got.copy()
    q2[0, 0, 1] = 0
    got2[0, 0, 1] = po.attend(q2[0, 0], sv.k[0], sv.v[0], 100, 0, sv.scale)[1]
    sv.check(q2, got2, tlm.FMT_F32)
    sv.close()


# ------------------------------------------------------- tables and batches --

@pytest.mark.parametrize("kv", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("tokens", [1, 3])
def test_entries_that_are_no_pages(ctx, kv, tokens):
    """Positions of a bad entry are not attended to, rows on one not appended; both are reported, once."""
    sv = Serving(ctx, 4, 2, 64, [200, 40, 90], tokens, 32, kv)
    sv.upload(*sv.pools(sv.starts + tokens))
    t = sv.tables.copy()
    t[0, 2], t[1, :], t[2, 0] = sv.pages, -5, 2 ** 31 - 1
    sv.batch.tables = ctx.array(t).ptr
    there = [np.repeat((t[s] >= 0) & (t[s] < sv.pages), 32) for s in range(3)]
    q = normal(sv)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, there, reported=True)
    with pytest.raises(tlm.TlmError) as e:
        sv.paged.status()
    assert e.value.code == tlm.TLM_ERR_RANGE and "no page" in str(e.value)
    sv.paged.status()
    kept = sv.kb.read(NP[kv]), sv.vb.read(NP[kv])
    t[:] = -1
    sv.batch.tables = ctx.array(t).ptr
    sv.paged.append(sv.batch, ctx.array(np.ones((3, tokens, 8, 64), np.float32)))
    with pytest.raises(tlm.TlmError):
        sv.paged.status()
    assert np.array_equal(sv.kb.read(NP[kv]), kept[0], equal_nan=True)
    assert np.array_equal(sv.vb.read(NP[kv]), kept[1], equal_nan=True)
    sv.close()


def test_rows_past_the_table_and_the_model_are_left_out(ctx):
    sv = Serving(ctx, 4, 2, 64, [62, 60, 5], 4, 32, counts=[4, 4, 4], max_tokens=70)
    sv.upload(*sv.pools([66, 64, 9]))
    b, q = sv.batch, normal(sv)
    # a table of two pages holds 64 positions: rows 2 and 3 of the first sequence are left out
    b.tables, b.table_width = ctx.array(sv.tables[:, :2].copy()).ptr, 2
    sv.rows = [2, 4, 4]
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, reported=True)
    with pytest.raises(tlm.TlmError) as e:
        sv.paged.status()
    assert e.value.code == tlm.TLM_ERR_RANGE and "left out" in str(e.value)
    # more rows than the batch has, and starts past everything
    b.tables, b.table_width = ctx.array(sv.tables).ptr, sv.width
    b.counts, b.starts = ctx.array(np.array([9, 4, 0], np.int32)).ptr, ctx.array(np.array([62, 2 ** 31 - 1, 5], np.int32)).ptr
    sv.rows = [4, 0, 0]
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, reported=True)
    before = sv.kb.read(np.float16)
    out = ctx.array(np.full((3, 4, 4 * 64), 77, np.float32))
    sv.paged.append(b, ctx.array(np.zeros((3, 4, 8, 64), np.float32)), out)
    got = out.read().reshape(3, 4, 256)
    assert np.all(got[0] == 0) and np.all(got[1:] == 77)
    after = sv.kb.read(np.float16)
    at = po.places(sv.tables[0], np.arange(62, 66), 2, 32, 64, 8, po.k_at)
    assert np.all(after[at] == 0)
    after[at] = before[at]
    assert np.array_equal(after, before, equal_nan=True)
    with pytest.raises(tlm.TlmError):
        sv.paged.status()
    sv.close()


def test_starts_past_everything_are_reported_by_either_call(ctx):
    sv = Serving(ctx, 4, 2, 64, [40, 3], 1, 32, counts=[1, 1], max_tokens=50)
    sv.upload(*sv.pools([41, 4]))
    q, x = normal(sv), np.zeros((2, 1, 8, 64), np.float32)
    for start in (50, 64, 2 ** 31 - 1):
        sv.batch.starts = ctx.array(np.array([start, 3], np.int32)).ptr
        sv.rows, sv.starts = [0, 1], np.array([start, 3], np.int32)
        sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, reported=True)
        with pytest.raises(tlm.TlmError) as e:
            sv.paged.status()
        assert e.value.code == tlm.TLM_ERR_RANGE
        sv.paged.append(sv.batch, ctx.array(x))
        with pytest.raises(tlm.TlmError):
            sv.paged.status()
        sv.paged.status()
        sv.upload(*sv.pools([0, 4]))
    sv.close()


@pytest.mark.parametrize("tokens", [1, 4])
def test_sequences_that_share_pages(ctx, tokens):
    """Two sequences with the same first pages (a cached prefix), then their own."""
    sv = Serving(ctx, 8, 2, 64, [150, 170], tokens, 32)
    sv.k[1][:128], sv.v[1][:128] = sv.k[0][:128], sv.v[0][:128]
    sv.tables[1, :4] = sv.tables[0, :4]
    sv.upload(*sv.pools(sv.starts + tokens))
    q = normal(sv)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32)
    sv.close()


def test_pools_past_32_bit_offsets(ctx):
    """Pages whose elements lie past 2^32 of a pool: two pools of 9 GB, of which three pages are used."""
    hkv, d, page = 8, 128, 256
    pages = (1 << 32) // (hkv * d * page) + 300
    sv = Serving(ctx, 16, hkv, d, [600], 2, page)
    one = hkv * d * page
    kb, vb = ctx.buffer(2 * one * pages), ctx.buffer(2 * one * pages)
    kp, vp = sv.pools(sv.starts + 2)
    table = np.array([[pages - 1, pages - 290, pages - 7]], np.int32)
    for i, p in enumerate(table[0]):
        src = int(sv.tables[0, i])
        for buf, host in ((kb, kp), (vb, vp)):
            a = np.ascontiguousarray(host[src * one:(src + 1) * one])
            tlm.check(tlm.lib().tlm_upload(ctx.ptr, ctypes.c_void_p(buf.ptr.value + 2 * one * int(p)),
                                           a.ctypes.data_as(ctypes.c_void_p), a.nbytes))
    sv.batch = sv.paged.batch(kb, vb, pages, ctx.array(table), 3, ctx.array(sv.starts), 1, 2)
    q = normal(sv)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32)
    x = sv.rng.standard_normal((1, 2, 32, d)).astype(np.float32)
    sv.paged.append(sv.batch, ctx.array(x))
    sv.paged.status()
    got = np.empty(one, np.float16)
    tlm.check(tlm.lib().tlm_download(ctx.ptr, got.ctypes.data_as(ctypes.c_void_p),
                                     ctypes.c_void_p(vb.ptr.value + 2 * one * int(table[0, 2])), got.nbytes))
    at = po.places([0, 0, 0], np.array([600, 601]), hkv, page, d, 8, po.v_at)
    assert np.array_equal(got[at], x[0, :, 24:].astype(np.float16))
    kb.free()
    vb.free()
    sv.close()


@pytest.mark.parametrize("shift", [4, 8, 12])
def test_rows_from_any_alignment(ctx, shift):
    """qkv, q and out from addresses that are no multiple of 16 bytes."""
    sv = Serving(ctx, 6, 2, 64, [70, 33], 3, 32)
    sv.upload(*sv.pools(sv.starts))

    class At:
        def __init__(self, a, fill=None):
            self.buf = ctx.buffer(a.nbytes + 16)
            self.ptr = ctypes.c_void_p(self.buf.ptr.value + shift)
            tlm.check(tlm.lib().tlm_upload(ctx.ptr, self.ptr, a.ctypes.data_as(ctypes.c_void_p), a.nbytes))
            self.like = a

        def read(self):
            out = np.empty_like(self.like)
            tlm.check(tlm.lib().tlm_download(ctx.ptr, out.ctypes.data_as(ctypes.c_void_p), self.ptr, out.nbytes))
            return out

    x = sv.rng.standard_normal((2, 3, 10, 64)).astype(np.float32)
    q, q0 = At(np.zeros((2, 3, 6, 64), np.float32)), ctx.buffer(2 * 3 * 6 * 64 * 4)
    kb, vb = sv.kb, sv.vb
    sv.paged.append(sv.batch, ctx.array(x), q0)
    k0, v0 = kb.read(np.float16), vb.read(np.float16)
    sv.paged.append(sv.batch, At(x), q)
    assert np.array_equal(q.read().ravel(), q0.read())
    assert np.array_equal(kb.read(np.float16), k0, equal_nan=True)
    assert np.array_equal(vb.read(np.float16), v0, equal_nan=True)
    for fmt in (tlm.FMT_F16, tlm.FMT_F32):
        a, b = ctx.buffer(2 * 3 * 6 * 64 * 4), At(np.zeros((2, 3, 6, 64), NP[fmt]))
        sv.paged.attention(sv.batch, q0, a, fmt)
        sv.paged.attention(sv.batch, q, b, fmt)
        assert np.array_equal(b.read().ravel(), a.read(NP[fmt])[:2 * 3 * 6 * 64])
    sv.close()


def test_refusals(ctx):
    sv = Serving(ctx, 4, 2, 64, [5], 1, 32)
    b = sv.upload(*sv.pools([6]))
    x, q, out = ctx.buffer(8 * 64 * 4), ctx.buffer(4 * 64 * 4), ctx.buffer(4 * 64 * 4)

    def refuse(code, call, *args):
        with pytest.raises(tlm.TlmError) as e:
            call(*args)
        assert e.value.code == code

    for field, value in (("k_pages", None), ("v_pages", None), ("tables", None), ("starts", None), ("num_pages", 0),
                         ("table_width", 0), ("seqs", 0), ("tokens", -1), ("k_pages", sv.kb.ptr.value + 2),
                         ("v_pages", sv.vb.ptr.value + 8)):
        keep = getattr(b, field)
        setattr(b, field, value)
        refuse(tlm.TLM_ERR_INVALID, sv.paged.append, b, x, q)
        refuse(tlm.TLM_ERR_INVALID, sv.paged.attention, b, q, out)
        setattr(b, field, keep)
    keep, b.v_pages = b.v_pages, sv.kb.ptr.value + 16  # the pools overlap
    refuse(tlm.TLM_ERR_INVALID, sv.paged.append, b, x, q)
    refuse(tlm.TLM_ERR_INVALID, sv.paged.attention, b, q, out)
    b.v_pages = keep
    b.seqs, b.tokens = 1 << 20, 1 << 20
    refuse(tlm.TLM_ERR_RANGE, sv.paged.append, b, x, q)
    refuse(tlm.TLM_ERR_RANGE, sv.paged.attention, b, q, out)
    b.seqs = b.tokens = 1
    refuse(tlm.TLM_ERR_INVALID, sv.paged.append, b, x, x)
    refuse(tlm.TLM_ERR_INVALID, sv.paged.attention, b, q, q)
    refuse(tlm.TLM_ERR_INVALID, sv.paged.attention, b, q, out, tlm.FMT_Q4)
    with pytest.raises(tlm.TlmError):
        tlm.Paged(ctx, 4, 2, 48, 100)
    for small in (dict(k_pages=sv.kb, num_pages=sv.pages + 1), dict(tables=ctx.buffer(4), table_width=2),
                  dict(starts=ctx.buffer(4), seqs=2), dict(counts=ctx.buffer(4), seqs=2)):
        whole = dict(k_pages=sv.kb, v_pages=sv.vb, num_pages=sv.pages, tables=ctx.buffer(64), table_width=1,
                     starts=ctx.buffer(64), seqs=1)
        refuse(tlm.TLM_ERR_INVALID, lambda: sv.paged.batch(**{**whole, **small}))
    sv.paged.append(b, x, q)
    sv.paged.status()
    sv.close()


def test_rope_tables_past_the_memory_are_refused(ctx):
    """512 GB of tables: refused before any is computed.  Without RoPE there are none."""
    free = ctx.memory()[0]
    with pytest.raises(tlm.TlmError) as e:
        tlm.Paged(ctx, 32, 8, 128, 1 << 30, inv_freq=np.ones(64, np.float32))
    assert e.value.code == tlm.TLM_ERR_OOM and "RoPE" in str(e.value)
    assert ctx.memory()[0] == free
    tlm.Paged(ctx, 32, 8, 128, 1 << 30).close()


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "tables", "starts", "counts"])
def test_results_over_what_the_batch_names_are_refused(ctx, name):
    """Every block reads the lengths and its pages for itself, while others write."""
    sv = Serving(ctx, 4, 2, 64, [5, 40], 2, 32, counts=[2, 1])
    b = sv.upload(*sv.pools([7, 41]))
    x, q, out = ctx.buffer(4 * 8 * 64 * 4), ctx.buffer(4 * 4 * 64 * 4), ctx.buffer(4 * 4 * 64 * 4)
    last = {"k_pages": sv.kb.nbytes, "v_pages": sv.vb.nbytes, "tables": 8 * sv.width, "starts": 8, "counts": 8}[name] - 4

    class At:
        def __init__(self, base, offset):
            self.ptr = ctypes.c_void_p(base + offset)

    def refuse(call, *args):
        with pytest.raises(tlm.TlmError) as e:
            call(*args)
        assert e.value.code == tlm.TLM_ERR_INVALID and "overlap" in str(e.value)

    at = At(getattr(b, name), last)
    refuse(sv.paged.append, b, x, at)
    for fmt in (tlm.FMT_F16, tlm.FMT_F32):
        refuse(sv.paged.attention, b, q, at, fmt)
    if name.endswith("pages"):
        refuse(sv.paged.append, b, at, q)
        for other in ("tables", "starts", "counts"):
            keep = getattr(b, other)
            setattr(b, other, getattr(b, name))
            refuse(sv.paged.append, b, x, q)
            setattr(b, other, keep)
    sv.paged.append(b, x, q)
    sv.paged.attention(b, q, out)
    sv.paged.status()
    sv.close()


def test_calls_allocate_nothing(ctx):
    sv = Serving(ctx, 8, 2, 64, [5000, 90, -1], 4, 32)
    sv.upload(*sv.pools([5004, 94, 0]))
    x, q = ctx.array(np.ones((3, 4, 12, 64), np.float32)), ctx.buffer(4 * 3 * 4 * 8 * 64)
    out = ctx.buffer(2 * 3 * 4 * 8 * 64)
    free = None
    for i in range(30):
        sv.paged.append(sv.batch, x, q)
        sv.paged.attention(sv.batch, q, out)
        ctx.sync()
        free = ctx.memory()[0] if i == 9 else free
    assert ctx.memory()[0] == free
    sv.paged.status()
    sv.close()


def test_two_contexts_at_once(ctx):
    """Calls of two contexts interleaved on their own streams, each with its own workspace."""
    other = tlm.Context(0)
    a = Serving(ctx, 8, 2, 64, [9000, 100], 1, 64, seed=1)
    b = Serving(other, 8, 2, 128, [12000], 2, 64, seed=2)
    qs, outs = [], []
    for sv in (a, b):
        sv.upload(*sv.pools([s + sv.tokens for s in sv.starts]))
        qs.append(normal(sv))
        outs.append([sv.ctx.buffer(4 * qs[-1].size) for _ in range(6)])
    qb = [sv.ctx.array(q) for sv, q in zip((a, b), qs)]
    for i in range(6):
        for sv, q, o in zip((a, b), qb, outs):
            sv.paged.attention(sv.batch, q, o[i], tlm.FMT_F32)
    for sv, q, o in zip((a, b), qs, outs):
        got = [x.read().reshape(q.shape) for x in o]
        sv.check(q, got[0], tlm.FMT_F32)
        assert all(np.array_equal(g, got[0]) for g in got)
        sv.close()
    other.close()
