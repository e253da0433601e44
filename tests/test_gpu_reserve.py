"""The reservation of pages against its plain form (more_oracle.py): whole numbers, all of them equal."""
import numpy as np
import pytest

import more_oracle as mo
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = tlm.Context(0)
    yield c
    c.close()


class Pool:
    """A handle and a pool's state on the host and on the device."""

    def __init__(self, ctx, n, width, pages, tokens, page=32, window=0, sinks=0, max_tokens=1 << 20, heads=1):
        self.ctx, self.n, self.width, self.pages, self.tokens, self.page = ctx, n, width, pages, tokens, page
        self.window, self.sinks, self.max_tokens = window, sinks, max_tokens
        self.paged = tlm.Paged(ctx, heads, 1, 32, max_tokens, page_tokens=page, sliding_window=window)
        if sinks:
            self.paged.set_sinks(sinks)
        self.tables, self.refs = np.full((n, width), -1, np.int32), np.zeros(pages, np.int32)

    def step(self, lengths, counts, in_place=False, slots=True):
        """One reservation; the state moves on."""
        c, n = self.ctx, self.n
        t, r = c.array(self.tables), c.array(self.refs)
        starts, sl = c.array(np.full(n, 77, np.int32)), c.array(np.full((n, self.tokens), 77, np.int64))
        ot = t if in_place else c.array(np.full((n, self.width), 77, np.int32))
        orf = r if in_place else c.array(np.full(self.pages, 77, np.int32))
        lengths = np.asarray(lengths, np.int32)
        counts = None if counts is None else np.asarray(counts, np.int32)
        req = self.paged.request(c.array(lengths), t, self.width, r, self.pages, starts, n, self.tokens,
                                 counts=None if counts is None else c.array(counts), slots=sl if slots else None,
                                 out_tables=ot, out_refs=orf)
        self.paged.reserve(req)
        got = (ot.read(np.int32).reshape(n, -1), orf.read(np.int32), starts.read(np.int32),
               sl.read(np.int64).reshape(n, -1))
        want = mo.reserve(self.tables, self.refs, lengths, counts, self.tokens, self.window, self.sinks, self.page,
                          self.max_tokens)
        if not slots:
            want[3][:] = 77
        for g, w, name in zip(got, want, ("tables", "refs", "starts", "slots")):
            assert np.array_equal(g, w), name
        if not in_place:
            assert np.array_equal(t.read(np.int32).reshape(n, -1), self.tables) and np.array_equal(r.read(np.int32), self.refs)
        bad, lost = want[4:]
        if bad or lost:
            with pytest.raises(tlm.TlmError) as e:
                self.paged.status()
            assert e.value.code == tlm.TLM_ERR_RANGE
            assert ("left out" in str(e.value)) == bad and ("no page" in str(e.value)) == lost
        else:
            self.paged.status()
        self.tables, self.refs = want[0], want[1]
        for b in {x.ptr.value: x for x in (t, r, starts, sl, ot, orf)}.values():
            b.free()
        return want[2]


@pytest.mark.parametrize("n,width,pages,tokens", [(1, 1, 1, 1), (1, 40, 50, 5), (7, 12, 60, 40), (64, 33, 900, 5),
                                                  (65, 64, 5000, 3), (300, 20, 4096, 2), (300, 20, 4097, 70),
                                                  (1100, 9, 9000, 1), (5, 2000, 20000, 3000)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 0), (70, 45), (1, 200)])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_of_a_server(ctx, n, width, pages, tokens, window, sinks, in_place):
    """Chats begin, go on, wait, end and give drafts back over a pool that others hold a part of; it runs short."""
    rng = np.random.default_rng([n, width, window])
    p = Pool(ctx, n, width, pages, tokens, 32, window, sinks)
    p.refs[rng.random(pages) < 0.3] = 2
    lengths = np.where(rng.random(n) < 0.8, 0, -1)
    for _ in range(6):
        counts = rng.integers(0, tokens + 1, n)
        starts = p.step(lengths, counts, in_place)
        served = starts >= 0
        lengths = np.where(served, lengths + rng.integers(0, np.maximum(counts, 0) + 1), lengths)
        lengths = np.where(rng.random(n) < 0.1, np.where(lengths < 0, 0, -1), lengths)
        lengths = np.minimum(lengths, width * 32)
    p.step(np.full(n, -1), None, in_place)
    assert np.all(p.tables == -1)
    p.paged.close()


@pytest.mark.parametrize("n,width,pages,tokens", [(1024, 32, 16384, 64), (1024, 32, 16385, 64), (1025, 31, 16384, 64),
                                                  (1024, 33, 16384, 64), (40, 100, 300, 3200), (2, 2100, 2300, 65537),
                                                  (3, 40, 1 << 20, 700), (3, 40, (1 << 20) + 5, 700),
                                                  (3, 40, 5000000, 700)])
@pytest.mark.parametrize("in_place", [True, False])
def test_sizes_where_the_kernels_change(ctx, n, width, pages, tokens, in_place):
    """The last size that one block takes and the first that it does not; the most pages whose returns are counted
    apart; more pages than 1024 blocks count."""
    rng = np.random.default_rng([n, width, pages])
    p = Pool(ctx, n, width, pages, tokens)
    p.refs[rng.random(pages) < 0.5] = 1
    lengths = np.zeros(n, np.int64)
    for _ in range(3):
        counts = rng.integers(0, tokens + 1, n)
        starts = p.step(lengths, counts, in_place)
        lengths = np.minimum(np.where(starts >= 0, lengths + counts, lengths), width * 32)
    p.paged.close()


@pytest.mark.parametrize("n,width,tokens", [(2, 5000, 4800), (3, 8193, 4800), (2, 20001, 4800), (2500, 1100, 1600)])
@pytest.mark.parametrize("quarter", [0, 1])
@pytest.mark.parametrize("in_place", [False, True])
def test_wide_tables(ctx, n, width, tokens, quarter, in_place):
    """Tables that sixteen waves share, and ones that their waves look at in several parts (widths that are no multiple
    of four, few waves for many sequences): pages held, lacking, given back and lost up to the last entry."""
    rng = np.random.default_rng([n, width, quarter])
    window, sinks = quarter * 8 * width, quarter * 70
    most = min(n, 12)  # with long tables; the others hold a few pages here and there
    pages = most * width + 8 * n + 17000
    ends = [((width - tokens // 32) * 32, tokens), (100, 5), (width * 32 - 20, 7), ((width - 1) * 32, 32)]
    for shift in range(4) if n < 4 else [0]:
        p = Pool(ctx, n, width, pages, tokens, 32, window, sinks)
        free = rng.permutation(pages)
        lengths, counts = rng.integers(-1, 60, n), rng.integers(0, 40, n)
        for s in range(n):
            where = np.arange(width) if s < most else np.concatenate([np.arange(2), rng.integers(2, width, 5), [width - 1]])
            p.tables[s, where], free = free[:where.size], free[where.size:]
        for s in range(most):
            kind = (s + shift) % 4
            lengths[s], counts[s] = ends[kind]
            if kind == 0:
                p.tables[s, width - tokens // 32:] = -1  # lacking, and some in between held
                p.tables[s, width - 7:width - 4], free = free[:3], free[3:]
            elif kind == 2:
                p.tables[s, width - 1] = -1  # holds positions
            elif kind == 3:
                p.tables[s, width - 1] = pages  # no page: lacking
        p.refs[:] = rng.random(pages) < 0.2  # others'
        np.add.at(p.refs, p.tables[(p.tables >= 0) & (p.tables < pages)], 1)
        starts = p.step(lengths, counts, in_place)
        for s in range(most):
            assert (starts[s] >= 0) == ((s + shift) % 4 != 2)
        lengths = np.where(starts >= 0, lengths + counts, lengths)
        lengths[(np.arange(n) + shift) % 4 == 3] = -1  # it ends
        p.step(np.minimum(lengths, width * 32), np.minimum(counts, 3), in_place)
        p.paged.close()


@pytest.mark.parametrize("page", [64, 1024])
def test_page_sizes(ctx, page):
    p = Pool(ctx, 6, 3, 20, 1500, page, 0, 0)
    p.step([0, 0, 0, 0, -1, 0], [1, page, page + 1, 2 * page, 5, 0])
    p.step([1, page, page + 1, page, 0, 7], [page - 1, 1, page, page, 1500, 1], True)
    p.paged.close()


def test_short_pools_serve_the_first(ctx):
    """Pages for some: the first that ask, and those that ask for none; the others keep what they have."""
    p = Pool(ctx, 8, 8, 10, 64, 32)
    starts = p.step([0] * 8, [64, 33, 32, 1, 64, 64, 1, 0])
    assert list(starts) == [0, 0, 0, 0, 0, 0, -1, -1]  # 2 + 2 + 1 + 1 + 2 + 2 of 10
    starts = p.step([64, 33, 32, 1, 64, 64, 0, 0], [1, 3, 1, 2, 0, 1, 1, 0])
    assert list(starts) == [-1, 33, -1, 1, -1, -1, -1, -1]
    starts = p.step([-1, 33, 32, 1, 64, 64, 0, 0], [1, 3, 1, 2, 0, 1, 1, 0])
    assert list(starts) == [-1, 33, 32, 1, -1, 64, -1, -1]
    p.paged.close()


def test_shared_pages_and_pins(ctx):
    """A prefix in three tables and one held by the caller: each count falls by one, nothing is handed out that is held."""
    p = Pool(ctx, 4, 4, 12, 4, 32)
    p.step([0, -1, -1, -1], [4, 0, 0, 0])
    p.refs[3] += 1  # the caller's
    p.tables[0, 1] = 5
    p.refs[5] = 4
    p.tables[1, :2] = p.tables[0, :2]
    p.tables[2, :2] = p.tables[0, :2]
    p.refs[p.tables[0, 0]] += 2
    p.step([64, 60, 64, -1], [4, 4, 4, 0])
    p.step([-1, 62, -1, 0], [4, 4, 4, 4], True)
    p.step([-1, -1, -1, 4], None)
    assert p.refs[5] == 1 and p.refs[3] == 1
    p.paged.close()


def test_rows_and_positions_out_of_range(ctx):
    """Counts above the batch's rows, rows past the table and the model's positions, entries that are no pages, and
    positions whose page is gone."""
    p = Pool(ctx, 7, 4, 40, 8, 32, max_tokens=100)
    starts = p.step([0, 0, 0, 0, 0, 0, 0], [9, 8, 1, 2, 2 ** 31 - 1, -5, 8])
    assert list(starts) == [0, 0, 0, 0, 0, -1, 0]
    p.tables[1, 2], p.tables[2, 3], p.tables[3, 0] = 40, -7, 2 ** 31 - 1
    p.step([8, 8, 1, 2, 8, -2 ** 31, 8], [1, 60, 8, 1, 8, 1, 8])
    p.step([96, 100, 127, 128, 2 ** 31 - 1, 200, 8], [8] * 7)
    p.paged.close()


def test_no_slots_and_no_counts(ctx):
    p = Pool(ctx, 5, 6, 30, 7, 32)
    p.step([0, 0, -1, 0, 0], None, slots=False)
    p.step([7, 3, 0, 7, 2], None, True)
    p.paged.close()


def test_refused(ctx):
    p = Pool(ctx, 4, 4, 9, 2).paged
    t, r, l, s = ctx.buffer(64), ctx.buffer(36), ctx.array(np.zeros(4, np.int32)), ctx.buffer(16)
    slots = ctx.buffer(8 * 8 + 8)
    ok = dict(lengths=l, tables=t, table_width=4, refs=r, num_pages=9, starts=s, seqs=4, tokens=2)

    def at(b, by):
        x = tlm.Buffer.__new__(tlm.Buffer)
        x.ctx, x.nbytes, x.ptr = ctx, 1 << 20, type(b.ptr)(b.ptr.value + by)
        return x

    wide = at(t, 0)  # a table as large as the counts: still not one for the other
    for change, code in ((dict(num_pages=0), tlm.TLM_ERR_INVALID), (dict(table_width=0), tlm.TLM_ERR_INVALID),
                         (dict(seqs=0), tlm.TLM_ERR_INVALID), (dict(tokens=0), tlm.TLM_ERR_INVALID),
                         (dict(out_tables=at(t, 4)), tlm.TLM_ERR_INVALID), (dict(out_refs=at(r, 4)), tlm.TLM_ERR_INVALID),
                         (dict(out_tables=at(r, 0)), tlm.TLM_ERR_INVALID), (dict(starts=at(l, 0)), tlm.TLM_ERR_INVALID),
                         (dict(out_refs=at(t, 0)), tlm.TLM_ERR_INVALID),
                         (dict(refs=wide, num_pages=16, out_refs=at(r, 0)), tlm.TLM_ERR_INVALID),
                         (dict(refs=at(r, 0), num_pages=16, out_tables=at(r, 0)), tlm.TLM_ERR_INVALID),
                         (dict(starts=at(t, 60)), tlm.TLM_ERR_INVALID), (dict(starts=at(r, 32)), tlm.TLM_ERR_INVALID),
                         (dict(slots=at(slots, 4)), tlm.TLM_ERR_INVALID), (dict(slots=at(t, 0)), tlm.TLM_ERR_INVALID)):
        with pytest.raises(tlm.TlmError) as e:
            p.reserve(p.request(**{**ok, **change}))
        assert e.value.code == code, change
    big = {k: at(ok[k], 0) for k in ("lengths", "tables", "refs", "starts")}
    for b in big.values():
        b.nbytes = 1 << 60
    for kw in (dict(seqs=1 << 20, tokens=5), dict(seqs=(1 << 20) + 1, tokens=1), dict(num_pages=(1 << 27) + 1),
               dict(table_width=(1 << 26) + 1)):
        with pytest.raises(tlm.TlmError) as e:
            p.reserve(p.request(**{**ok, **big, **kw}))
        assert e.value.code == tlm.TLM_ERR_RANGE, kw
    p.close()


def test_many_sequences_and_pages(ctx):
    """2^18 sequences over a pool of 2^21 pages, most of them held: every one that lacks a page gets the next free."""
    n, width, pages = 1 << 18, 2, 1 << 21
    rng = np.random.default_rng(0)
    p = tlm.Paged(ctx, 1, 1, 32, 64, page_tokens=32)
    refs = (rng.random(pages) < 0.85).astype(np.int32)
    lengths = np.where(rng.random(n) < 0.9, 0, -1).astype(np.int32)
    b = [ctx.array(lengths), ctx.array(np.full((n, width), -1, np.int32)), ctx.array(refs), ctx.array(np.full(n, 77, np.int32)),
         ctx.array(np.full(n, 77, np.int64))]
    p.reserve(p.request(b[0], b[1], width, b[2], pages, b[3], n, 1, slots=b[4]))
    tables, got, starts, slots = b[1].read(np.int32).reshape(n, width), b[2].read(np.int32), b[3].read(np.int32), b[4].read(np.int64)
    p.status()
    free = np.nonzero(refs == 0)[0]
    served = np.cumsum(lengths >= 0) * (lengths >= 0)
    assert served.max() <= free.size
    want = np.where(served > 0, free[np.maximum(served - 1, 0)], -1)
    assert np.array_equal(tables[:, 0], want) and np.all(tables[:, 1] == -1)
    assert np.array_equal(starts, np.where(served > 0, 0, -1)) and np.array_equal(slots, np.where(want >= 0, want * 32, -1))
    refs[want[want >= 0]] = 1
    assert np.array_equal(got, refs)
    for x in b:
        x.free()
    p.close()
