"""A server's steps as its program makes them: pages reserved from the lengths, rows appended to an 8-bit cache (and an
fp16 one), attention with a window and sinks, the head's logits under penalties, biases and masks, drafts verified.  Each
operator's results are checked against its plain form on what the operators before it left on the device."""
import numpy as np
import pytest

import more_oracle as mo
import paged_oracle as po
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


@pytest.mark.parametrize("kv,window,sinks", [(tlm.FMT_F8, 0, 0), (tlm.FMT_F8, 48, 8), (tlm.FMT_F16, 48, 8)])
def test_steps(kv, window, sinks):
    ctx = tlm.Context(0)
    rng = np.random.default_rng(5)
    n, t, hq, hkv, d, page, width, pages, vocab, hist = 5, 4, 4, 2, 64, 32, 8, 26, 501, 160
    inv = (1e4 ** (-np.arange(0, d, 2) / d)).astype(np.float32)
    paged = tlm.Paged(ctx, hq, hkv, d, width * page, page_tokens=page, inv_freq=inv, sliding_window=window, kv_fmt=kv)
    if sinks:
        paged.set_sinks(sinks)
    head = tlm.Linear(ctx, tlm.FMT_F16, (rng.standard_normal((vocab, hq * d)) * 0.2).astype(np.float16).view(np.uint16))
    i32 = lambda *shape: ctx.array(np.zeros(shape, np.int32))  # noqa: E731
    tables, refs, starts = ctx.array(np.full((n, width), -1, np.int32)), i32(pages), i32(n)
    slots = ctx.buffer(8 * n * t)
    kp, vp = (ctx.array(np.full(pages * paged.page_bytes(), 0x7F, np.uint8)) for _ in range(2))
    lens, counts, q, att = i32(n), i32(n), ctx.buffer(4 * n * t * hq * d), ctx.buffer(2 * n * t * hq * d)
    logits, ruled = ctx.buffer(4 * n * t * vocab), ctx.buffer(4 * n * t * vocab)
    said, history, drafts = i32(n), i32(n, hist), i32(n, t - 1)
    acc, ids = i32(n), i32(n, t)
    masks = rng.integers(0, 2 ** 32, (n, t, -(-vocab // 32)), dtype=np.uint64).astype(np.uint32)
    bias_ids, biases = rng.integers(0, vocab, (n, 3)).astype(np.int32), rng.standard_normal((n, 3)).astype(np.float32)
    rep, fre, pre = (rng.uniform(0.1, 1.4, n).astype(np.float32) for _ in range(3))
    # what the program keeps from step to step
    request = paged.request(lens, tables, width, refs, pages, starts, n, t, counts=counts, slots=slots)
    batch = paged.batch(kp, vp, pages, tables, width, starts, n, t, counts=counts)
    rules = tlm.logit_rules(logits, n, t, vocab, out=ruled, counts=counts, history=history, history_width=hist,
                            history_counts=said, drafts=drafts, repetition=ctx.array(rep), frequency=ctx.array(fre),
                            presence=ctx.array(pre), bias_ids=ctx.array(bias_ids), biases=ctx.array(biases),
                            bias_width=3, masks=ctx.array(masks))
    length, text = np.zeros(n, np.int32), [[int(rng.integers(vocab))] for _ in range(n)]
    length[4] = -1  # joins later
    cache = {name: [np.zeros((width * page, hkv, d)) for _ in range(n)] for name in "kv"}
    host_t, host_r = np.full((n, width), -1, np.int32), np.zeros(pages, np.int32)
    served = 0
    for turn in range(26):
        want = rng.integers(1, t + 1, n).astype(np.int32)
        if turn == 9:
            length[1], text[1] = -1, [1]  # ends, and its pages go to the one that joins
            length[4], text[4] = 0, [2]
        if turn == 15:
            length[1] = 0
        draft = rng.integers(0, vocab, (n, t - 1)).astype(np.int32)
        x = rng.standard_normal((n, t, hq + 2 * hkv, d)).astype(np.float32)
        hist_ids = np.zeros((n, hist), np.int32)
        for s in range(n):
            hist_ids[s, :len(text[s])] = text[s]
        lens.write(length), counts.write(want), drafts.write(draft), history.write(hist_ids)
        said.write(np.array([len(s) for s in text], np.int32))
        qkv = ctx.array(x)
        att.write(np.full(n * t * hq * d, 0.25, np.float16))

        paged.reserve(request)
        paged.append(batch, qkv, q)
        paged.attention(batch, q, att)
        head.rows(att, n * t, logits)
        tlm.adjust_logits(ctx, rules)
        tlm.verify_drafts(ctx, ruled, n, t, vocab, acc, ids, drafts=drafts, counts=counts, temperature=0.0)
        paged.status()

        host_t, host_r, go, want_slots, bad, lost = mo.reserve(host_t, host_r, length, want, t, window, sinks, page, width * page)
        assert not bad and not lost
        assert np.array_equal(tables.read(np.int32).reshape(n, -1), host_t) and np.array_equal(refs.read(np.int32), host_r)
        assert np.array_equal(starts.read(np.int32), go) and np.array_equal(slots.read(np.int64).reshape(n, t), want_slots)
        pools = {"k": kp.read(np.uint8), "v": vp.read(np.uint8)}
        qh, a = q.read().reshape(n, t, hq, d), att.read(np.float16).reshape(n, t, hq, d)
        for s in range(n):
            r = int(want[s]) if go[s] >= 0 else 0
            assert np.all(a[s, r:] == 0.25)
            if not r:
                continue
            served += 1
            end = int(length[s]) + r
            pos = np.arange(end)
            pos = pos[host_t[s, pos // page] >= 0]
            rot = po.rope(x[s, :r, :hq + hkv], np.arange(length[s], end), inv)
            assert np.all(np.abs(qh[s, :r] - rot[:, :hq]) <= 8 * EPS * np.abs(x[s, :r, :hq]).max())
            for name, new in (("k", rot[:, hq:]), ("v", x[s, :r, hq + hkv:])):
                if kv == tlm.FMT_F8:
                    where = mo.k8_at if name == "k" else mo.v8_at
                    scale = pools[name].view(np.float32)[mo.scales_at(host_t[s], pos, hkv, page, d)].astype(np.float64)
                    val = mo.CODES[pools[name][mo.places8(host_t[s], pos, hkv, page, d, where)]] * scale[..., None]
                    # half a step of the value, or of the smallest codes of its scale
                    near = np.abs(new) * 2.0 ** -4 * 1.01 + 2.0 ** -10 * scale[-r:, :, None] * 1.01
                else:
                    val = pools[name].view(np.float16)[po.places(host_t[s], pos, hkv, page, d, 8, po.k_at if name == "k" else po.v_at)]
                    val, near = val.astype(np.float64), np.abs(new) * 2.0 ** -11 * 1.01 + 2.0 ** -24
                assert np.all(np.abs(val[-r:] - new) <= near)
                cache[name][s][pos] = val
            for j in range(r):
                p = int(length[s]) + j
                keys = mo.visible(p, window, sinks)
                ref = mo.attend(qh[s, j], cache["k"][s], cache["v"][s], keys, d ** -0.5)
                big = float((np.abs(cache["k"][s][keys]).repeat(2, 1) * np.abs(qh[s, j])).sum(-1).max()) * d ** -0.5
                tol = (2 * (d / 4 + 8) * max(big, 1) + 200) * EPS * np.abs(cache["v"][s][keys]).max() + 2.0 ** -11 * np.abs(ref)
                assert np.all(np.abs(a[s, j] - ref) <= tol + 2.0 ** -25)
        lg, lr = logits.read().reshape(n, t, vocab), ruled.read().reshape(n, t, vocab)
        ref, size = mo.adjust(lg, want, hist_ids, [len(s) for s in text], draft, rep, fre, pre, bias_ids, biases, masks, lr)
        fine = np.isfinite(ref)
        assert np.array_equal(np.isfinite(lr), fine)
        assert np.all(np.abs(lr[fine] - ref[fine]) <= 7 * EPS * size[fine] + 1e-30)
        accepted, tokens = po.verify(lr, draft, want, None, 0)
        got_acc, got_ids = acc.read(np.int32), ids.read(np.int32).reshape(n, t)
        for s in range(n):
            assert got_acc[s] == accepted[s] and np.array_equal(got_ids[s], tokens[s])
            if go[s] < 0:
                continue
            length[s] += 1 + accepted[s]
            text[s] += [int(v) for v in tokens[s, :accepted[s] + 1] if v >= 0]
            if length[s] + t > width * page or len(text[s]) + t > hist:
                length[s], text[s] = -1, [0]
    assert served > 80
    paged.close()
    head.close()
    ctx.close()


def test_two_contexts_at_once():
    """Two programs' calls in turn, nothing waits between them: each one's results are what it gets alone."""
    rng = np.random.default_rng(3)
    n, hq, hkv, d, page, width, pages, vocab = 3, 8, 2, 64, 32, 64, 200, 3000
    x = rng.standard_normal((2, n, 40, hq + 2 * hkv, d)).astype(np.float32)
    logits = rng.standard_normal((2, n, vocab)).astype(np.float32)
    ids = rng.integers(0, vocab, (2, n, 50)).astype(np.int32)

    def begin(ctx, k):
        p = tlm.Paged(ctx, hq, hkv, d, width * page, page_tokens=page, sliding_window=1500, kv_fmt=tlm.FMT_F8)
        p.set_sinks(5)
        z = lambda *shape: ctx.array(np.zeros(shape, np.int32))  # noqa: E731
        b = dict(tables=ctx.array(np.full((n, width), -1, np.int32)), refs=z(pages), starts=z(n), q=ctx.buffer(4 * n * 40 * hq * d),
                 out=ctx.array(np.zeros((n, 40, hq * d), np.float32)), x=ctx.array(x[k]), logits=ctx.array(logits[k]),
                 kp=ctx.array(np.zeros(pages * p.page_bytes(), np.uint8)), vp=ctx.array(np.zeros(pages * p.page_bytes(), np.uint8)))
        lengths = [ctx.array(np.array([40 * i, 40 * i - 3 if i else 0, 40 * i], np.int32)) for i in range(46)]
        rules = tlm.logit_rules(b["logits"], n, 1, vocab, history=ctx.array(ids[k]), history_width=50,
                                frequency=ctx.array(np.full(n, 0.5, np.float32)))
        return p, b, lengths, rules

    def step(ctx, state, i):
        p, b, lengths, rules = state
        p.reserve(p.request(lengths[i], b["tables"], width, b["refs"], pages, b["starts"], n, 40))
        batch = p.batch(b["kp"], b["vp"], pages, b["tables"], width, b["starts"], n, 40)
        p.append(batch, b["x"], b["q"])
        p.attention(batch, b["q"], b["out"], tlm.FMT_F32)
        tlm.adjust_logits(ctx, rules)

    def end(state):
        p, b, _, _ = state
        p.status()
        r = [b["tables"].read(np.int32), b["refs"].read(np.int32), b["kp"].read(np.uint8), b["vp"].read(np.uint8),
             b["out"].read(), b["logits"].read()]
        p.close()
        return r

    alone = []
    for k in range(2):
        ctx = tlm.Context(0)
        s = begin(ctx, k)
        for i in range(46):
            step(ctx, s, i)
        alone.append(end(s))
        ctx.close()
    both = [tlm.Context(0), tlm.Context(0)]
    states = [begin(c, k) for k, c in enumerate(both)]
    for i in range(46):
        for c, s in zip(both, states):
            step(c, s, i)
    for s, want in zip(states, alone):
        for got, w in zip(end(s), want):
            assert np.array_equal(got.view(np.uint8), w.view(np.uint8))
    for c in both:
        c.close()


def test_a_step_of_idle_slots():
    """No sequence has rows: nothing is written, nothing reported."""
    ctx = tlm.Context(0)
    for kv in (tlm.FMT_F8, tlm.FMT_F16):
        p = tlm.Paged(ctx, 4, 2, 64, 256, page_tokens=32, sliding_window=40, kv_fmt=kv)
        p.set_sinks(3)
        kp = ctx.array(np.full(4 * p.page_bytes(), 7, np.uint8))
        vp = ctx.array(np.full(4 * p.page_bytes(), 7, np.uint8))
        b = p.batch(kp, vp, 4, ctx.array(np.full((70, 8), -1, np.int32)), 8, ctx.array(np.full(70, -1, np.int32)), 70, 2)
        q, out = ctx.array(np.full((70, 2, 256), 5, np.float32)), ctx.array(np.full((70, 2, 256), 6, np.float32))
        p.append(b, ctx.array(np.full((70, 2, 512), 1, np.float32)), q)
        p.attention(b, q, out, tlm.FMT_F32)
        p.status()
        assert np.all(kp.read(np.uint8) == 7) and np.all(vp.read(np.uint8) == 7)
        assert np.all(q.read() == 5) and np.all(out.read() == 6)
        p.close()
    ctx.close()
