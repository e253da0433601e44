"""The paged cache of 8-bit values and windows with sinks against 64-bit forms (more_oracle.py), at the sizes, scales
and masks where they can go wrong.  The pools hold NaN codes and NaN scales (fp16, fp32: NaN) wherever no
sequence's position lies, tables hold -1 wherever no page is needed.

Tolerances.  Append: a rotated element is off by 4 * 2^-24 of |a| + |b| (test_gpu_paged.py); its code is the
nearest to some value within that, so it is off by half a step of the codes there (2^-4 of the value, 2^-10 of the
scale below 2^-6 of it) and the rounding of the element.  V and unrotated K are the nearest codes exactly.
Positions that were there are coded again from their codes, exactly as the formula says.  Attention: as for the
other caches (test_gpu_paged.py), over the values that the codes and scales stand for."""
import numpy as np
import pytest

import more_oracle as mo
import paged_oracle as po
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HALF = {tlm.FMT_F16: 2.0 ** -11, tlm.FMT_F32: 2.0 ** -24}
NP = {tlm.FMT_F16: np.float16, tlm.FMT_F32: np.float32}
F8 = tlm.FMT_F8


@pytest.fixture(scope="module")
def ctx():
    c = tlm.Context(0)
    yield c
    c.close()


class Serving:
    """Sequences with caches of random rows: on the host their values (and, of 8 bits, codes and scales' exponents),
    on the device pools and tables."""

    def __init__(self, ctx, hq, hkv, d, lengths, tokens, page=32, kv=F8, window=0, sinks=0, counts=None, seed=0,
                 rotary=None, spare=2, spread=2, max_tokens=None, scale=0.0):
        self.ctx, self.hq, self.hkv, self.d, self.page, self.kv = ctx, hq, hkv, d, page, kv
        self.window, self.sinks = window, sinks
        rng = self.rng = np.random.default_rng([seed, hq, d, page, tokens, window, sinks])
        self.n, self.tokens, self.starts = len(lengths), tokens, np.array(lengths, np.int32)
        self.counts = None if counts is None else np.array(counts, np.int32)
        self.rows = [0 if s < 0 else tokens if counts is None else min(max(counts[i], 0), tokens)
                     for i, s in enumerate(lengths)]
        self.ends = [s + r if r else 0 for s, r in zip(lengths, self.rows)]
        used = [mo.pages_in_use(s, r, window, sinks, page) if r else [] for s, r in zip(lengths, self.rows)]
        self.width = max(1, max((u[-1] + 1 for u in used if u), default=1))
        self.pages = sum(map(len, used)) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((self.n, self.width), -1, np.int32)
        at = 0
        for s, u in enumerate(used):
            self.tables[s, u] = order[at:at + len(u)]
            at += len(u)
        self.used = used
        rd = d if rotary is None else rotary
        self.inv = (1e4 ** (-np.arange(0, rd, 2) / rd)).astype(np.float32) if rd else None
        self.scale = scale or d ** -0.5
        self.paged = tlm.Paged(ctx, hq, hkv, d, max_tokens or self.width * page, page_tokens=page, inv_freq=self.inv,
                               rotary_dim=rd or None, sliding_window=window, kv_fmt=kv, attn_scale=scale)
        if sinks:
            self.paged.set_sinks(sinks)
        self.k, self.v, self.codes, self.exps = [], [], {"k": [], "v": []}, {"k": [], "v": []}
        for e in self.ends:
            for name in ("k", "v"):
                if kv == F8:
                    c = rng.integers(0, 256, (e, hkv, d)).astype(np.uint8)
                    c[c & 127 >= 0x78] &= 0x87  # up to 240, no NaN: some codes of every exponent
                    x = np.repeat(rng.integers(-7 - spread, -7 + spread + 1, (-(-e // 32), hkv)), 32, 0)[:e]
                    self.codes[name].append(c)
                    self.exps[name].append(x)
                    val = mo.CODES[c] * 2.0 ** x[..., None]
                else:
                    val = rng.standard_normal((e, hkv, d)).astype(NP[kv])
                (self.k if name == "k" else self.v).append(val)

    def positions(self, s, upto):
        """Positions of the sequence that lie in a page of its table."""
        p = np.arange(upto)
        return p[np.isin(p // self.page, self.used[s])]

    def pools(self, upto):
        """Host pools with positions [0, upto[s]) of every sequence as far as it has pages, NaN elsewhere."""
        out = []
        for name, where in (("k", mo.k8_at), ("v", mo.v8_at)):
            if self.kv == F8:
                size = mo.page_bytes(self.hkv, self.page, self.d)
                pool = np.full((self.pages, size), 0x7F, np.uint8)
                pool[:, self.hkv * self.page * self.d:].view(np.uint32)[:] = 0x7FC00000
                pool = pool.reshape(-1)
            else:
                pool = np.full(self.pages * self.hkv * self.page * self.d, np.nan, NP[self.kv])
            for s in range(self.n):
                pos = self.positions(s, upto[s])
                if not pos.size:
                    continue
                if self.kv == F8:
                    pool[mo.places8(self.tables[s], pos, self.hkv, self.page, self.d, where)] = self.codes[name][s][pos]
                    at = mo.scales_at(self.tables[s], pos, self.hkv, self.page, self.d)
                    pool.view(np.float32)[at] = 2.0 ** self.exps[name][s][pos].astype(np.float64)
                else:
                    e = 4 if self.kv == tlm.FMT_F32 else 8
                    at = po.places(self.tables[s], pos, self.hkv, self.page, self.d, e, po.k_at if name == "k" else po.v_at)
                    pool[at] = (self.k if name == "k" else self.v)[s][pos]
            out.append(pool)
        return out

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

    def check(self, q, got, out_fmt, exact_nan=False):
        if self.counts is not None and np.any((self.counts > self.tokens) & (self.starts >= 0)):
            with pytest.raises(tlm.TlmError) as e:  # a count above the batch's rows: reported, those computed
                self.paged.status()
            assert e.value.code == tlm.TLM_ERR_RANGE
        else:
            self.paged.status()
        for s in range(self.n):
            assert np.all(got[s, self.rows[s]:] == 77), f"rows behind sequence {s}"
            for j in range(self.rows[s]):
                pos = int(self.starts[s]) + j
                keys = mo.visible(pos, self.window, self.sinks)
                ref = mo.attend(q[s, j], self.k[s], self.v[s], keys, self.scale)
                kk = np.abs(self.k[s][keys].astype(np.float64)).repeat(self.hq // self.hkv, 1)
                big = max(1.0, float((kk * np.abs(q[s, j])).sum(-1).max()) * self.scale)
                mv = float(np.nanmax(np.abs(self.v[s][keys].astype(np.float64))))
                tol = (2 * (self.d / 4 + 8) * big + keys.size / 16 + 96) * EPS * mv + HALF[out_fmt] * np.abs(ref)
                g = got[s, j].astype(np.float64)
                if exact_nan:
                    assert np.array_equal(np.isnan(g), np.isnan(ref)), f"NaN of sequence {s} row {j}"
                    g, ref, tol = np.nan_to_num(g), np.nan_to_num(ref), np.nan_to_num(tol)
                err = np.abs(g - ref)
                assert np.all(err <= tol + 2.0 ** -25), f"sequence {s} row {j}: {np.nanmax(err - tol)} over {err.max()}"

    def close(self):
        self.paged.close()


def normal(sv):
    return sv.rng.standard_normal((sv.n, sv.tokens, sv.hq, sv.d)).astype(np.float32)


def attend(sv, out_fmt=tlm.FMT_F32):
    sv.upload(*sv.pools(sv.ends))
    q = normal(sv)
    sv.check(q, sv.attention(q, out_fmt), out_fmt)
    sv.close()


# ------------------------------------------------------------------- append --

def append(sv, x=None, want_q=True):
    """One append against the formula; the pools' other bytes stay."""
    kp, vp = sv.pools(np.maximum(sv.starts, 0) * (np.array(sv.rows) > 0))
    sv.upload(kp, vp)
    if x is None:
        x = sv.rng.standard_normal((sv.n, sv.tokens, sv.hq + 2 * sv.hkv, sv.d)).astype(np.float32)
    q = sv.ctx.array(np.full((sv.n, sv.tokens, sv.hq, sv.d), 77, np.float32))
    sv.paged.append(sv.batch, sv.ctx.array(x), q if want_q else None)
    got_q = q.read().reshape(sv.n, sv.tokens, sv.hq, sv.d)
    got = {"k": sv.kb.read(np.uint8), "v": sv.vb.read(np.uint8)}
    sv.paged.status()
    h, hkv = sv.hq, sv.hkv
    finite = np.where(np.isfinite(x), x, 0)
    touched = {"k": np.zeros(kp.size, bool), "v": np.zeros(kp.size, bool)}
    for s in range(sv.n):
        r = sv.rows[s]
        assert np.all(got_q[s, r if want_q else 0:] == 77)
        if not r:
            continue
        p0 = int(sv.starts[s])
        pos = p0 + np.arange(r)
        half = 0 if sv.inv is None else sv.inv.size
        with np.errstate(invalid="ignore"):
            rot = po.rope(x[s, :r, :h + hkv], pos, sv.inv)
        mag = np.abs(finite[s, :r, :h + hkv]).astype(np.float64)
        mag[..., :2 * half] = np.concatenate([mag[..., :half] + mag[..., half:2 * half]] * 2, -1)
        if want_q:
            e = np.abs(got_q[s, :r] - rot[:, :h])
            assert np.all((e <= 4 * EPS * mag[:, :h]) | ~np.isfinite(rot[:, :h])), f"q of {s}"
        off = 4 * EPS * mag[:, h:]
        if sv.inv is None:
            off[:] = 0
        for name, new, tol, where in (("k", rot[:, h:], off, mo.k8_at),
                                      ("v", x[s, :r, h + hkv:].astype(np.float64), np.zeros_like(off), mo.v8_at)):
            at = mo.places8(sv.tables[s], pos, hkv, sv.page, sv.d, where)
            sat = mo.scales_at(sv.tables[s], pos, hkv, sv.page, sv.d)
            scale = got[name].view(np.float32)[sat].astype(np.float64)
            for b in range(p0 // 32, (p0 + r - 1) // 32 + 1):
                rows = np.nonzero(pos // 32 == b)[0]
                size = np.where(np.isfinite(new[rows]), np.abs(new[rows]), 0)
                lo, hi = np.maximum(size - tol[rows], 0).max((0, 2)), (size + tol[rows]).max((0, 2))
                held = np.arange(b * 32, max(p0, b * 32))
                for g in range(hkv):
                    e = [mo.exponent(lo[g]), mo.exponent(hi[g])]
                    if held.size:
                        old = int(sv.exps[name][s][held[0], g])
                        e = [max(old, v) for v in e]
                    assert scale[rows[0], g] in (2.0 ** e[0], 2.0 ** e[1]), (name, s, b, g)
                if held.size:  # coded again
                    hat = mo.places8(sv.tables[s], held, hkv, sv.page, sv.d, where)
                    ratio = 2.0 ** sv.exps[name][s][held].astype(np.float64) / scale[rows[0]]
                    want = mo.encode(mo.CODES[sv.codes[name][s][held]] * ratio[..., None])
                    assert np.array_equal(got[name][hat], want), f"what {name} of {s} had"
                    touched[name][hat] = True
            code = got[name][at]
            val = mo.CODES[code] * scale[..., None]
            assert np.array_equal(np.isnan(val), ~np.isfinite(new)), f"NaN of {name} of {s}"
            big = np.clip(np.nan_to_num(new, posinf=0, neginf=0), -448 * 2.0 ** 31, 448 * 2.0 ** 31)
            bound = np.minimum(mo.step((np.abs(big) + tol) / scale[..., None]) * scale[..., None] / 2, np.inf) + tol
            err = np.abs(np.nan_to_num(val) - big)
            assert np.all(err <= bound), f"{name} of {s}: {np.max(err - bound)}"
            if not tol.any():
                fine = np.isfinite(new)
                assert np.array_equal(code[fine], mo.encode(big / scale[..., None])[fine]), f"codes of {name} of {s}"
            touched[name][at] = True
            for i in range(4):
                touched[name][4 * sat + i] = True
    for name, was in (("k", kp), ("v", vp)):
        assert np.array_equal(got[name][~touched[name]], was[~touched[name]]), f"bytes of no new position in {name}"
    sv.close()


@pytest.mark.parametrize("hq,hkv,d,page", [(14, 2, 64, 64), (24, 8, 128, 32), (4, 4, 32, 128), (6, 1, 96, 32)])
@pytest.mark.parametrize("tokens", [1, 5, 45])
def test_append(ctx, hq, hkv, d, page, tokens):
    counts = [tokens, 1, max(1, tokens - 3), 0, tokens]
    append(Serving(ctx, hq, hkv, d, [0, 63, 30, 12, -1], tokens, page, counts=counts))


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 64, 100, 300])
@pytest.mark.parametrize("start", [0, 1, 16, 31, 45])
def test_append_at_block_edges(ctx, tokens, start):
    append(Serving(ctx, 4, 2, 64, [start, start + 7], tokens, 32, counts=[tokens, max(1, tokens - 2)], rotary=0))


@pytest.mark.parametrize("rotary", [0, 2, 20, 32, 48])
@pytest.mark.parametrize("tokens", [1, 70])
def test_append_partial_rotary_and_no_q(ctx, rotary, tokens):
    append(Serving(ctx, 3, 1, 64, [9, 40], tokens, 64, rotary=rotary))
    append(Serving(ctx, 3, 1, 64, [9, 40], tokens, 64, rotary=rotary), want_q=False)


@pytest.mark.parametrize("rotary", [0, 16, 64, 112, 128])
@pytest.mark.parametrize("tokens", [3, 40])
def test_append_partial_rotary_of_wide_heads(ctx, rotary, tokens):
    append(Serving(ctx, 4, 2, 128, [9, 40], tokens, 64, rotary=rotary))


@pytest.mark.parametrize("hq,hkv,d", [(40, 40, 32), (48, 3, 64), (33, 33, 128)])
@pytest.mark.parametrize("tokens", [1, 5, 33])
def test_append_many_heads(ctx, hq, hkv, d, tokens):
    append(Serving(ctx, hq, hkv, d, [30, 5], tokens, 32))


def test_append_far_positions(ctx):
    append(Serving(ctx, 2, 1, 128, [100000, 99999, 65535, 131071], 2, 128, window=40, max_tokens=1 << 18))


@pytest.mark.parametrize("old", [-32, -20, -7, 0, 20, 31])
@pytest.mark.parametrize("size", [1e-12, 2.0 ** -7, 1.0, 2.0 ** 20, 2.0 ** 45])
def test_append_scales(ctx, old, size):
    """Rows far below, near and far above what their block holds, to the ends of the scales' range."""
    sv = Serving(ctx, 2, 1, 64, [40, 33, 63], 3, 32, rotary=0, counts=[3, 1, 2])
    for name in ("k", "v"):
        for x in sv.exps[name]:
            x[:] = old
    x = (sv.rng.standard_normal((3, 3, 4, 64)) * size).astype(np.float32)
    append(sv, x)


@pytest.mark.parametrize("tokens", [1, 33])
def test_append_every_code_and_the_halves_between(ctx, tokens):
    """Each code's value, the points halfway to the next and their neighbours, subnormal codes among them; zeros of
    both signs and rows of zeros."""
    v = mo.CODES[:127].astype(np.float32)
    mid = ((v[:-1] + v[1:]) / 2).astype(np.float32)
    near = [np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))]
    vals = np.concatenate([v, mid, *near, -v, -mid, [0.0, -0.0]]).astype(np.float32)
    sv = Serving(ctx, 1, 1, 64, [0, 20], tokens, 32, rotary=0)
    x = np.zeros((2, tokens, 3, 64), np.float32)
    flat = np.resize(vals, x.size).reshape(x.shape)
    x[:, :, 1:] = flat[:, :, 1:] * np.float32(2.0 ** -5)
    x[..., 1:, 0] = 448 * 2.0 ** -5  # the scale is what it is
    if tokens > 1:
        x[1, -1] = 0
    append(sv, x)
    append(Serving(ctx, 1, 1, 64, [0, 32], tokens, 32, rotary=0), np.zeros_like(x))


def test_append_values_that_are_not_finite(ctx):
    """NaN and infinities become NaN codes, and the scale is the others'."""
    sv = Serving(ctx, 1, 1, 64, [0, 20, 31], 4, 32, rotary=0)
    x = sv.rng.standard_normal((3, 4, 3, 64)).astype(np.float32)
    x[0, 1, 1, 5], x[1, 2, 2, 7], x[2, 0, 1, 0], x[2, 3, 2, 63] = np.nan, np.inf, -np.inf, np.nan
    append(sv, x)


def test_append_one_by_one_equals_the_values(ctx):
    """40 tokens appended one at a time, their size growing and shrinking: each code within a rounding for every time
    that its block's scale grew."""
    n, d, page = 40, 64, 32
    sv = Serving(ctx, 2, 1, d, [n - 1], 1, page, rotary=0, spare=0)
    sv.upload(*sv.pools([0]))
    x = sv.rng.standard_normal((n, 4, d)).astype(np.float32) * (2.0 ** sv.rng.integers(-6, 7, n)).astype(np.float32)[:, None, None]
    for p in range(n):
        sv.batch.starts = (keep := ctx.array(np.array([p], np.int32))).ptr
        sv.paged.append(sv.batch, ctx.array(x[p]))
        ctx.sync()
    sv.paged.status()
    pos = np.arange(n)
    for buf, where, rows in ((sv.kb, mo.k8_at, x[:, 2]), (sv.vb, mo.v8_at, x[:, 3])):
        pool = buf.read(np.uint8)
        scale = pool.view(np.float32)[mo.scales_at(sv.tables[0], pos, 1, page, d)].astype(np.float64)[..., None]
        got = (mo.CODES[pool[mo.places8(sv.tables[0], pos, 1, page, d, where)]] * scale)[:, 0]
        for b in (slice(0, 32), slice(32, 40)):
            assert np.all(scale[b] == 2.0 ** mo.exponent(np.abs(rows[b]).max()))
            # each rounding is half a step of what it rounds, of the last scale's at most; it grew 12 times at most
            err = np.abs(got[b] - rows[b])
            coarse = 2.0 ** -10 * scale[b][:, 0]
            assert np.all(err <= np.abs(rows[b]) * 2.0 ** -4 + 2 * coarse)
    sv.close()


# ---------------------------------------------------------------- attention --

@pytest.mark.parametrize("out_fmt", [tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(14, 2, 64, 64), (24, 8, 128, 32), (4, 4, 32, 128), (16, 1, 96, 32)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_attention_shapes(ctx, hq, hkv, d, page, out_fmt, tokens):
    attend(Serving(ctx, hq, hkv, d, [0, 15, 31, 32, 200, -1, 517], tokens, page,
                   counts=[tokens, tokens, 1, tokens, 2, 1, tokens]), out_fmt)


@pytest.mark.parametrize("start", [0, 1, 15, 16, 30, 31, 32, 33, 63, 64, 255, 256, 257, 1000, 2047, 2048])
def test_attention_lengths(ctx, start):
    attend(Serving(ctx, 8, 2, 64, [start], 1, 64))


@pytest.mark.parametrize("tokens", [2, 5, 16, 17, 40, 130])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 64), (24, 8, 128), (16, 1, 128)])
def test_attention_drafts_and_chunks(ctx, tokens, hq, hkv, d):
    attend(Serving(ctx, hq, hkv, d, [0, 29, 300], tokens, 32, counts=[tokens, tokens, max(1, tokens - 1)]))


@pytest.mark.parametrize("tokens", [1, 5])
def test_attention_one_long_cache_among_short_ones(ctx, tokens):
    attend(Serving(ctx, 8, 2, 128, [20000, 3, 700], tokens, 256))


@pytest.mark.parametrize("n", [65, 300, 500])
def test_attention_of_many_sequences(ctx, n):
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in rng.integers(0, 60, n)]
    for s in (1, 63, 64, n - 1):
        lengths[s] = 2500 + 7 * s
    lengths[5] = -1
    attend(Serving(ctx, 4, 2, 64, lengths, 1, 64))


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("spread", [12, 24])
def test_attention_over_scales_far_apart(ctx, spread, tokens):
    """V's scales up to 2^48 apart, K's few: a row whose weights lie where V is small is as exact as its weights, and
    the large values weigh what they weigh."""
    sv = Serving(ctx, 4, 2, 64, [700, 90, 1500], tokens, 32, spread=spread)
    for s in range(sv.n):
        sv.exps["k"][s] = np.clip(sv.exps["k"][s], -8, -6)
        sv.k[s] = mo.CODES[sv.codes["k"][s]] * 2.0 ** sv.exps["k"][s][..., None]
    attend(sv)


def test_a_certain_key_where_v_is_small(ctx):
    """The row's weight lies on one key of a block whose V is 2^-50 of the others': its V, exactly."""
    sv = Serving(ctx, 4, 2, 64, [900, 900], 2, 64, scale=1.0)
    for s, at in ((0, 70), (1, 870)):
        sv.exps["v"][s][:] = 25
        sv.exps["v"][s][at // 32 * 32:at // 32 * 32 + 32] = -25
        sv.v[s] = mo.CODES[sv.codes["v"][s]] * 2.0 ** sv.exps["v"][s][..., None]
        sv.codes["k"][s][:] = 0x20
        sv.codes["k"][s][at] = 0x77
        sv.exps["k"][s][:] = 0
        sv.k[s] = mo.CODES[sv.codes["k"][s]] * 1.0
    sv.upload(*sv.pools(sv.ends))
    q = np.abs(normal(sv)) + 1
    got = sv.attention(q, tlm.FMT_F32).astype(np.float64)
    sv.paged.status()
    for s, at in ((0, 70), (1, 870)):
        want = sv.v[s][at].repeat(2, 0)
        assert np.all(np.abs(got[s] - want) <= 2.0 ** -20 * np.abs(want)), s
    sv.close()


@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 24, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(ctx, size, sign):
    """Scores past what a 32-bit number holds in whole steps, V's scales far apart: the best key's V, and of keys with
    the same score their mean."""
    sv = Serving(ctx, 4, 2, 64, [300, 40], 3, 32, scale=1.0, spread=20)
    best = [(7, 290), (7, 35)]
    for s in range(2):
        sv.exps["k"][s][:] = 0
        sv.codes["k"][s][:] = 0
        sv.codes["k"][s][..., 0] = 0x38 if sign > 0 else 0x40  # 1, or 2
        for at in best[s]:
            sv.codes["k"][s][at, :, 0] = 0x40 if sign > 0 else 0x38
        sv.k[s] = mo.CODES[sv.codes["k"][s]] * 1.0
    sv.upload(*sv.pools(sv.ends))
    q = np.zeros((2, 3, 4, 64), np.float32)
    q[..., 0] = sign * size * (1 + np.arange(4) / 8)
    got = sv.attention(q, tlm.FMT_F32).astype(np.float64)
    sv.paged.status()
    for s in range(2):
        two = sv.v[s][list(best[s])]
        want, mv = two.mean(0).repeat(2, 0), np.abs(two).max(0).repeat(2, 0)
        assert np.all(np.abs(got[s] - want) <= 2.0 ** -20 * mv + 2.0 ** -39 * np.abs(two).max()), s
    sv.close()


def test_attention_over_what_append_wrote(ctx):
    """Appended, then attended, in one stream; the cache read back is what is attended to."""
    sv = Serving(ctx, 8, 2, 64, [0, 40, 100, 31], 37, 32, rotary=64)
    sv.upload(*sv.pools(np.maximum(sv.starts, 0)))
    x = sv.rng.standard_normal((4, 37, 12, 64)).astype(np.float32)
    q = ctx.buffer(4 * 4 * 37 * 8 * 64)
    sv.paged.append(sv.batch, ctx.array(x), q)
    out = ctx.array(np.full((4, 37, 8 * 64), 77, np.float32))
    sv.paged.attention(sv.batch, q, out, tlm.FMT_F32)
    got, qh = out.read().reshape(4, 37, 8, 64), q.read().reshape(4, 37, 8, 64)
    for buf, where, keep in ((sv.kb, mo.k8_at, sv.k), (sv.vb, mo.v8_at, sv.v)):
        pool = buf.read(np.uint8)
        for s in range(4):
            pos = np.arange(sv.ends[s])
            scale = pool.view(np.float32)[mo.scales_at(sv.tables[s], pos, 2, 32, 64)].astype(np.float64)
            keep[s] = mo.CODES[pool[mo.places8(sv.tables[s], pos, 2, 32, 64, where)]] * scale[..., None]
    sv.check(qh, got, tlm.FMT_F32)
    sv.close()


@pytest.mark.parametrize("tokens", [5, 40])
def test_pools_past_32_bits(ctx, tokens):
    """Pages that begin past 2^32 bytes of the pools: appended, attended to, read back."""
    hq, hkv, d, page, pages = 8, 8, 128, 1024, 4200
    p = tlm.Paged(ctx, hq, hkv, d, 4 * page, page_tokens=page, kv_fmt=F8)
    size = p.page_bytes()
    assert 4100 * size > 1 << 32
    kb, vb = ctx.buffer(pages * size), ctx.buffer(pages * size)
    tables, starts = np.array([[4199, -1], [4101, 4150]], np.int32), np.array([0, 0], np.int32)
    rng = np.random.default_rng(tokens)
    x = rng.standard_normal((2, tokens, hq + 2 * hkv, d)).astype(np.float32)
    b = p.batch(kb, vb, pages, ctx.array(tables), 2, ctx.array(starts), 2, tokens)
    q, out = ctx.buffer(4 * 2 * tokens * hq * d), ctx.buffer(4 * 2 * tokens * hq * d)
    p.append(b, ctx.array(x), q)
    p.attention(b, q, out, tlm.FMT_F32)
    p.status()
    got, rows = out.read().reshape(2, tokens, hq, d).astype(np.float64), {}
    assert np.array_equal(q.read().reshape(2, tokens, hq, d), x[:, :, :hq])  # no rotation here
    for s in range(2):
        for name, buf, new, where in (("k", kb, x[s, :, hq:2 * hq], mo.k8_at), ("v", vb, x[s, :, 2 * hq:], mo.v8_at)):
            at = tlm.Buffer.__new__(tlm.Buffer)  # the sequence's page
            at.ctx, at.nbytes, at.ptr = ctx, size, type(buf.ptr)(buf.ptr.value + int(tables[s, 0]) * size)
            one, pos = at.read(np.uint8), np.arange(tokens)
            scale = one.view(np.float32)[mo.scales_at([0], pos, hkv, page, d)].astype(np.float64)
            code = one[mo.places8([0], pos, hkv, page, d, where)]
            assert np.array_equal(code, mo.encode(new / scale[..., None]))
            rows[name] = mo.CODES[code] * scale[..., None]
        for j in range(tokens):
            ref = mo.attend(x[s, j, :hq], rows["k"], rows["v"], np.arange(j + 1), d ** -0.5)
            assert np.all(np.abs(got[s, j] - ref) <= 2.0 ** -16 * np.abs(rows["v"]).max())
    kb.free()
    vb.free()
    p.close()


def test_nan_reaches_only_the_rows_that_see_it(ctx):
    """A NaN in the last positions' V: rows before it are as they would be without, rows that see it are NaN there."""
    sv = Serving(ctx, 4, 2, 64, [60, 10], 6, 32)
    for s, (p, h, c) in ((0, (64, 1, 9)), (1, (15, 0, 63))):
        sv.codes["v"][s][p, h, c] = 0xFF
        sv.v[s][p, h, c] = np.nan
    sv.upload(*sv.pools(sv.ends))
    q = normal(sv)
    sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32, exact_nan=True)
    sv.close()


@pytest.mark.parametrize("kv,window,sinks", [(F8, 0, 0), (F8, 1060, 40), (tlm.FMT_F16, 1060, 40)])
@pytest.mark.parametrize("n,hkv", [(100, 4), (400, 1)])
def test_attention_of_many_sequences_of_one_length(ctx, n, hkv, kv, window, sinks):
    """So many that they stay whole, whatever their length; a few idle ones and a short one among them."""
    lengths = [1090 + s % 40 for s in range(n)]
    lengths[3], lengths[n - 1] = -1, 2
    attend(Serving(ctx, hkv, hkv, 32, lengths, 1, 64, kv, window=window, sinks=sinks))


# -------------------------------------------------------------------- sinks --

@pytest.mark.parametrize("sinks", [1, 4, 31, 32, 33, 100, 700])
@pytest.mark.parametrize("window", [1, 31, 32, 100])
@pytest.mark.parametrize("kv", [F8, tlm.FMT_F16, tlm.FMT_F32])
def test_sinks(ctx, kv, window, sinks):
    """The pages between the sinks and the window are given back: -1 in the tables, NaN in the pool."""
    attend(Serving(ctx, 8, 2, 64, [0, 3, window - 1, window + 45, 1500], 2, 32, kv, window=window, sinks=sinks,
                   counts=[2, 1, 2, 2, 2]))


@pytest.mark.parametrize("tokens", [6, 40, 150, 400])
@pytest.mark.parametrize("window,sinks", [(20, 4), (20, 130), (64, 64), (333, 5)])
@pytest.mark.parametrize("kv", [F8, tlm.FMT_F16])
def test_sinks_of_prompts(ctx, kv, window, sinks, tokens):
    """Chunks of prompts from the first token on, behind their sinks, and across the end of them."""
    attend(Serving(ctx, 4, 1, 64, [0, 50, 129, 800], tokens, 64, kv, window=window, sinks=sinks))


@pytest.mark.parametrize("kv", [F8, tlm.FMT_F16, tlm.FMT_F32])
@pytest.mark.parametrize("window,sinks", [(3000, 1000), (5000, 4), (40, 6000)])
def test_sinks_in_several_chunks(ctx, kv, window, sinks):
    attend(Serving(ctx, 8, 2, 128, [20000, 3, 9000], 2, 256, kv, window=window, sinks=sinks))


@pytest.mark.parametrize("n", [70, 400])
def test_sinks_of_many_sequences(ctx, n):
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in np.exp(rng.uniform(0, np.log(3000), n))]
    lengths[7] = -1
    attend(Serving(ctx, 2, 1, 64, lengths, 1, 32, tlm.FMT_F16, window=200, sinks=70))


def test_sinks_change_and_end(ctx):
    """0 sinks are none; more than the positions are all of them; a handle without a window refuses them."""
    sv = Serving(ctx, 4, 2, 64, [500], 2, 32, tlm.FMT_F16, window=40, sinks=600)
    sv.upload(*sv.pools(sv.ends))
    q = normal(sv)
    for sinks in (600, 0, 5, 1 << 30):
        sv.paged.set_sinks(sinks)
        sv.sinks = sinks
        sv.check(q, sv.attention(q, tlm.FMT_F32), tlm.FMT_F32)
    for sinks in (-1, (1 << 30) + 1):
        with pytest.raises(tlm.TlmError) as e:
            sv.paged.set_sinks(sinks)
        assert e.value.code == tlm.TLM_ERR_INVALID
    sv.close()
    whole = tlm.Paged(ctx, 4, 2, 64, 100, page_tokens=32)
    whole.set_sinks(0)
    with pytest.raises(tlm.TlmError) as e:
        whole.set_sinks(4)
    assert e.value.code == tlm.TLM_ERR_INVALID and "window" in str(e.value)
    whole.close()


# ------------------------------------------------------------- what is refused --

def test_pages_that_are_none_are_reported(ctx):
    """A sequence whose table names no page of the pool: nothing of it is appended, its positions are not attended to."""
    sv = Serving(ctx, 4, 2, 64, [40, 70], 2, 32)
    sv.tables[0, 1] = sv.pages
    kp, vp = sv.pools([32, 70])
    sv.upload(kp, vp)
    x = sv.rng.standard_normal((2, 2, 8, 64)).astype(np.float32)
    sv.paged.append(sv.batch, ctx.array(x))
    with pytest.raises(tlm.TlmError) as e:
        sv.paged.status()
    assert e.value.code == tlm.TLM_ERR_RANGE and "no page" in str(e.value)
    got = sv.kb.read(np.uint8)
    at = mo.places8(sv.tables[1], [70, 71], 2, 32, 64, mo.k8_at)
    assert not np.array_equal(got[at], kp[at])
    mine = mo.places8(sv.tables[0], range(32), 2, 32, 64, mo.k8_at)
    assert np.array_equal(got[mine], kp[mine])
    q = normal(sv)
    out = sv.attention(q, tlm.FMT_F32)
    with pytest.raises(tlm.TlmError):
        sv.paged.status()
    for j in range(2):
        ref = mo.attend(q[0, j], sv.k[0], sv.v[0], np.arange(32), sv.scale)
        assert np.all(np.abs(out[0, j] - ref) <= 2.0 ** -18 * np.abs(sv.v[0][:32]).max())
    sv.close()


def test_results_over_the_scales_are_refused(ctx):
    """A pool of 8-bit values is its codes and its scales."""
    p = tlm.Paged(ctx, 4, 2, 64, 256, page_tokens=32, kv_fmt=F8)
    size = p.page_bytes()
    pool, other = ctx.buffer(4 * size + 4096), ctx.buffer(4 * size)
    ints = ctx.array(np.zeros(16, np.int32))
    b = p.batch(pool, other, 4, ints, 4, ctx.array(np.zeros(1, np.int32)), 1)
    last = tlm.Buffer.__new__(tlm.Buffer)
    last.ctx, last.nbytes, last.ptr = ctx, 1 << 20, type(pool.ptr)(pool.ptr.value + 4 * size - 4)
    q = ctx.buffer(4 * 4 * 64)
    for call in (lambda: p.attention(b, q, last, tlm.FMT_F32), lambda: p.append(b, last, q),
                 lambda: p.append(b, ctx.buffer(4 * 8 * 64), last)):
        with pytest.raises(tlm.TlmError) as e:
            call()
        assert e.value.code == tlm.TLM_ERR_INVALID and "overlap" in str(e.value)
    p.close()


def test_other_caches_are_not_of_8_bits(ctx):
    with pytest.raises(tlm.TlmError) as e:
        tlm.Attention(ctx, 4, 2, 64, 100, inv_freq=np.ones(32, np.float32), kv_fmt=F8)
    assert e.value.code == tlm.TLM_ERR_INVALID and "paged" in str(e.value)
    d = tlm.ModelDesc(256, 512, 1, 4, 2, 64, 1000, 64, 64, 0, tlm.FMT_F16, tlm.FMT_F16, tlm.FMT_F16, F8)
    with pytest.raises(tlm.TlmError) as e:
        tlm.Model(ctx, d, np.ones(32, np.float32))
    assert e.value.code == tlm.TLM_ERR_INVALID and "paged" in str(e.value)
