"""Verification of drafted tokens against its 64-bit definition (paged_oracle.verify):
whole numbers, so every one has to be the definition's."""
import numpy as np
import pytest

import paged_oracle as po
import three_llm_amd.tlm as tlm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = tlm.Context(0)
    yield c
    c.close()


def check(ctx, logits, drafts, uniforms, temp, counts=None, draft_logits=None):
    n, t, v = logits.shape
    acc, ids = ctx.array(np.full(n, -7, np.int32)), ctx.array(np.full((n, t), -7, np.int32))
    opt = lambda a, dt: None if a is None else ctx.array(np.asarray(a, dt))  # noqa: E731
    tlm.verify_drafts(ctx, ctx.array(np.asarray(logits, np.float32)), n, t, v, acc, ids, drafts=opt(drafts, np.int32),
                      draft_logits=opt(draft_logits, np.float32), counts=opt(counts, np.int32),
                      uniforms=opt(uniforms, np.float32), temperature=temp)
    a, i = acc.read(np.int32), ids.read(np.int32).reshape(n, t)
    ra, ri = po.verify(logits, drafts, counts, uniforms, temp, draft_logits)
    assert np.array_equal(a, ra), (a, ra)
    assert np.array_equal(i, ri), (i, ri)
    return a, i


def inputs(n, t, v, seed=0, spread=2.0, by="lookup", close=0.5):
    rng = np.random.default_rng([seed, n, t, v])
    logits = (rng.standard_normal((n, t, v)) * spread).astype(np.float32)
    u = rng.random((n, t), np.float32)
    q = None
    about = logits[:, :-1]
    if by == "model" and t > 1:
        q = about = (about + rng.standard_normal(about.shape) * close).astype(np.float32)
    drafts = (about / 0.8 + rng.gumbel(size=about.shape) * (1.0 if by == "model" else 0.3)).argmax(-1) if t > 1 else None
    return logits, drafts, u, q


@pytest.mark.parametrize("v", [1, 2, 63, 64, 255, 2047, 2048, 2049, 4099, 32000])
@pytest.mark.parametrize("t", [1, 2, 5])
@pytest.mark.parametrize("by", ["lookup", "model"])
def test_vocabularies(ctx, v, t, by):
    logits, drafts, u, q = inputs(6, t, v, by=by)
    for temp in (0.0, 0.7, 1.0):
        check(ctx, logits, drafts, u, temp, draft_logits=q)


@pytest.mark.parametrize("by", ["lookup", "model"])
def test_large_vocabulary_many_sequences(ctx, by):
    logits, drafts, u, q = inputs(12, 4, 151936, by=by)
    check(ctx, logits, drafts, u, 0.8, counts=[4, 1, 0, 3, 2, 4, 4, -3, 4, 1, 2, 4], draft_logits=q)


@pytest.mark.parametrize("n,v", [(64, 3000), (65, 4097), (200, 2049), (4097, 40), (9000, 7)])
@pytest.mark.parametrize("by", ["lookup", "model"])
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_many_sequences_of_all_counts(ctx, n, v, by, temp):
    """More sequences than a wave's lanes, than a launch's counters; idle ones in between."""
    logits, drafts, u, q = inputs(n, 3, v, by=by)
    counts = np.random.default_rng(n).integers(-1, 4, n)
    check(ctx, logits, drafts, u, temp, counts=counts, draft_logits=q)


def test_flat_distribution_draws_the_definition_s_token(ctx):
    """Every token equally likely but for noise: the sums decide."""
    logits, _, u, _ = inputs(48, 1, 128256, spread=0.05)
    check(ctx, logits, None, u, 1.0)


def test_most_rows(ctx):
    logits, drafts, u, _ = inputs(3, 64, 500, spread=6.0)
    drafts[:] = logits[:, :-1].argmax(-1)
    a, _ = check(ctx, logits, drafts, np.zeros_like(u), 0.5)
    assert np.all(a == 63)
    check(ctx, logits, drafts, u, 0.0)
    check(ctx, logits, drafts, u, 0.3, counts=[64, 63, 2])


@pytest.mark.parametrize("v", [131073, 524287, 524288])
@pytest.mark.parametrize("by", ["lookup", "model"])
def test_largest_vocabularies(ctx, v, by):
    """Rows of more than 64 chunks, so several to a lane; the last sequence's tokens lie at the end of its rows."""
    logits, drafts, u, q = inputs(6, 2, v, by=by)
    logits[5, :, :v - 40] -= np.float32(60)
    drafts[4, 0] = v - 1
    for temp in (0.0, 0.8):
        check(ctx, logits, drafts, u, temp, draft_logits=q)


def test_most_rows_of_a_draft_model(ctx):
    logits, drafts, u, q = inputs(5, 64, 2500, by="model", close=0.05)
    check(ctx, logits, drafts, u * np.float32(0.5), 0.8, counts=[64, 63, 9, 33, 8], draft_logits=q)
    check(ctx, logits, drafts, u, 0.8, draft_logits=q)


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 0.5])
@pytest.mark.parametrize("by", ["lookup", "model"])
def test_ends_of_the_random_numbers(ctx, u, by):
    logits, drafts, x, q = inputs(8, 3, 5000, by=by)
    check(ctx, logits, drafts, np.full_like(x, u), 0.9, draft_logits=q)


def test_borders_that_are_exact(ctx):
    """Equal logits: every weight is one, u * v lands on borders exactly, and the next token is drawn."""
    v = 4096
    u = (np.arange(64, dtype=np.float32) * 64 / v).reshape(64, 1)
    _, ids = check(ctx, np.zeros((64, 1, v), np.float32), None, u, 1.0)
    assert np.array_equal(ids[:, 0], np.arange(64) * 64)


@pytest.mark.parametrize("temp", [0.0, 1.0])
@pytest.mark.parametrize("by", ["lookup", "model"])
def test_masked_entries_and_rows(ctx, temp, by):
    """-inf, LOWEST_FLOAT and NaN take no part; rows of nothing else give -1; an infinite score takes all."""
    logits, drafts, u, q = inputs(7, 3, 3000, by=by)
    logits[0, :, 1::2] = -np.inf
    logits[1, :, ::3] = np.nan
    logits[2, 0] = -np.inf
    logits[3, 1] = np.float32(po.LOWEST)
    logits[4, 0, 100] = np.inf
    logits[5, 0] = -np.inf
    logits[5, 0, 2999] = -1e30
    logits[6, 0, :2999] = np.nan
    drafts[4, 0] = 100
    drafts[5, 0] = 2999
    if q is not None:
        q[0, 0] = -np.inf
        q[1, 1, 5:] = np.nan
        q[6] = np.nan
    check(ctx, logits, drafts, u, temp, draft_logits=q)


@pytest.mark.parametrize("temp", [0.0, 1.0])
@pytest.mark.parametrize("by", ["lookup", "model"])
def test_drafts_outside_the_vocabulary(ctx, temp, by):
    logits, drafts, u, q = inputs(4, 3, 700, by=by)
    drafts[:, 0] = [-1, 700, 2 ** 31 - 1, -2 ** 31]
    a, _ = check(ctx, logits, drafts, u, temp, draft_logits=q)
    assert np.all(a == 0)


def test_a_draft_that_holds_nearly_all(ctx):
    """p(x) = 1 - 1e-5 or so and u above it: what is left is drawn from, to its last digits."""
    logits, drafts, u, _ = inputs(6, 2, 20000, spread=1.0)
    for s, top in enumerate((20.0, 22.0, 24.0, 18.0, 26.0, 200.0)):
        drafts[s, 0] = 777 * (s + 1)
        logits[s, 0, drafts[s, 0]] = top
    u[:, 0] = 1.0 - 2.0 ** -24
    check(ctx, logits, drafts, u, 1.0)


def test_target_and_draft_model_the_same(ctx):
    """p = q: every draft stands, as u < 1."""
    logits, drafts, u, _ = inputs(5, 4, 9000)
    a, _ = check(ctx, logits, drafts, u, 1.0, draft_logits=logits[:, :-1].copy())
    assert np.all(a == 3)


@pytest.mark.parametrize("shift", [0.5, -3.0, 1e-3])
@pytest.mark.parametrize("v", [700, 9000])
def test_nothing_but_rounding_beside_a_draft_model(ctx, shift, v):
    """q's logits are p's and a constant, and no draft can stand: what is left of p - q is rounding or nothing, and some
    token of the vocabulary is drawn all the same."""
    n = 40
    logits, _, u, _ = inputs(n, 2, v)
    acc, ids = ctx.buffer(4 * n), ctx.buffer(8 * n)
    tlm.verify_drafts(ctx, ctx.array(logits), n, 2, v, acc, ids, drafts=ctx.array(np.full((n, 1), -1, np.int32)),
                      draft_logits=ctx.array(logits[:, :1] + np.float32(shift)), uniforms=ctx.array(u), temperature=1.0)
    assert np.all(acc.read(np.int32) == 0)
    first = ids.read(np.int32).reshape(n, 2)[:, 0]
    assert np.all((first >= 0) & (first < v))


@pytest.mark.parametrize("temp", [1e-9, 1e-6, 0.01, 50.0, 1e30])
def test_temperatures(ctx, temp):
    logits, drafts, u, q = inputs(5, 3, 4000, by="model")
    check(ctx, logits, drafts, u, temp, draft_logits=q)
    check(ctx, logits, drafts, u, temp)


def test_frequencies_follow_the_target(ctx):
    """20000 drafts of a draft model and what is emitted for them: the first token is the target's, whatever the
    draft's distribution.  A frequency of p is off by sqrt(p (1 - p) / 20000): five of those."""
    rng = np.random.default_rng(5)
    n, v = 20000, 8
    p, q = rng.standard_normal(v).astype(np.float32), rng.standard_normal(v).astype(np.float32)
    pp, pq = po.softmax(p, 1.0)[0], po.softmax(q, 1.0)[0]
    drafts = rng.choice(v, size=(n, 1), p=pq).astype(np.int32)
    logits = np.broadcast_to(p, (n, 2, v)).copy()
    acc, ids = ctx.buffer(4 * n), ctx.buffer(8 * n)
    tlm.verify_drafts(ctx, ctx.array(logits), n, 2, v, acc, ids, drafts=ctx.array(drafts),
                      draft_logits=ctx.array(np.broadcast_to(q, (n, 1, v)).copy()),
                      uniforms=ctx.array(rng.random((n, 2), np.float32)), temperature=1.0)
    got = np.bincount(ids.read(np.int32).reshape(n, 2)[:, 0], minlength=v) / n
    assert np.all(np.abs(got - pp) <= 5 * np.sqrt(pp * (1 - pp) / n))


def test_refusals(ctx):
    b = ctx.buffer(1 << 16)

    def refuse(code, *args, **kw):
        with pytest.raises(tlm.TlmError) as e:
            tlm.verify_drafts(ctx, *args, **kw)
        assert e.value.code == code and "TLMVerify" in str(e.value)

    refuse(tlm.TLM_ERR_INVALID, b, 0, 1, 10, b, b, uniforms=b)
    refuse(tlm.TLM_ERR_INVALID, b, 1, 0, 10, b, b, uniforms=b)
    refuse(tlm.TLM_ERR_INVALID, b, 1, 1, 0, b, b, uniforms=b)
    refuse(tlm.TLM_ERR_INVALID, b, 1, 65, 2, b, b, drafts=b, uniforms=b)
    refuse(tlm.TLM_ERR_INVALID, b, 1, 1, 524289, b, b, uniforms=b)
    refuse(tlm.TLM_ERR_RANGE, b, 4096, 64, 524288, b, b, drafts=b, uniforms=b)  # the workspace
    refuse(tlm.TLM_ERR_INVALID, b, 1, 2, 10, b, b, uniforms=b)
    refuse(tlm.TLM_ERR_INVALID, b, 1, 2, 10, b, b, drafts=b)
    for temp in (-0.5, float("nan"), float("inf")):
        refuse(tlm.TLM_ERR_INVALID, b, 1, 1, 10, b, b, uniforms=b, temperature=temp)
    refuse(tlm.TLM_ERR_RANGE, b, 1 << 20, 2, 10, b, b, drafts=b, uniforms=b)


@pytest.mark.parametrize("name", ["logits", "draft_logits", "drafts", "counts", "uniforms", "accepted"])
def test_results_over_an_input_are_refused(ctx, name):
    # a sequence's results are written while others' inputs are still read
    S, T, V = 3, 4, 10
    held = {k: ctx.buffer(4 * S * T * V) for k in ("logits", "draft_logits", "drafts", "counts", "uniforms", "accepted",
                                                   "out_tokens")}
    held["out_tokens"] = held[name]

    def call(temperature):
        b = dict(held)
        tlm.verify_drafts(ctx, b.pop("logits"), S, T, V, b.pop("accepted"), b.pop("out_tokens"), temperature=temperature,
                          **b)

    with pytest.raises(tlm.TlmError) as e:
        call(1.0)
    assert e.value.code == tlm.TLM_ERR_INVALID and "overlap" in str(e.value)
    if name in ("draft_logits", "uniforms"):  # not read there
        held["counts"].write(np.zeros(S, np.int32))
        call(0.0)
