"""The 8-bit cache's layout and scales, the pages in use, and the refusals, on the host; the plain forms
(more_oracle.py) against differences of their own."""
import ctypes
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from test_host import header_struct_fields
from test_paged import buffer, refused, says
import more_oracle as mo
import three_llm_amd.tlm as tlm

SHIM = """
#include "tlm_paged.h"
using namespace tlm;
extern "C" int k_at(int t, int d, int D) { return paged8_k_at(t, d, D); }
extern "C" int v_at(int t, int d, int D) { return paged8_v_at(t, d, D); }
extern "C" int exponent(uint32_t top) { return paged8_exponent(top); }
extern "C" int exponent_of(uint32_t scale) { return paged8_exponent_of(scale); }
extern "C" void use(int start, int rows, int window, int sinks, int shift, int* out) {
  const PagedUse u = paged_use(start, rows, window, sinks, shift);
  out[0] = u.sink, out[1] = u.first, out[2] = u.end;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The kernels' own arithmetic, built for the host."""
    d = tmp_path_factory.mktemp("more")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", str(ROOT / "three-llm_amd" / "csrc"), "-o",
                    str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("cname,pytype", [("tlm_paged_request", tlm.PagedRequest), ("tlm_logit_rules", tlm.LogitRules)])
def test_structs_match_the_header(cname, pytype):
    assert [f for f, _ in pytype._fields_] == header_struct_fields(cname)


def test_codes():
    """Every code is its own nearest; halves between two go to the even one; a little off them to the nearer."""
    v = mo.CODES
    whole = [c for c in range(256) if c & 127 != 127]
    assert np.array_equal(mo.encode(v[whole]), np.array(whole, np.uint8))
    assert v[126] == 448 and v[8] == 2.0 ** -6 and v[1] == 2.0 ** -9
    for c in range(126):
        mid = (v[c] + v[c + 1]) / 2
        assert mo.encode(mid) == c + (c & 1) and mo.encode(-mid) == (c + (c & 1)) | 128
        assert mo.encode(mid * (1 - 1e-9)) == c and mo.encode(mid * (1 + 1e-9)) == c + 1


def test_codes_under_a_larger_scale():
    """Coded again, values from 2^-6 of the new scale on are exact; below it some are not, up to 2^-13.8 of a largest
    magnitude that the scale is the least for."""
    whole = mo.CODES[[c for c in range(256) if c & 127 != 127]]
    largest = np.nextafter(np.float32(224), np.float32(225))
    assert mo.exponent(float(largest)) == 0 and mo.exponent(224.0) == -1
    inexact = 0.0
    for by in range(1, 64):
        v = whole * 2.0 ** -by
        again = mo.CODES[mo.encode(v)]
        assert np.array_equal(again[np.abs(v) >= 2.0 ** -6], v[np.abs(v) >= 2.0 ** -6])
        inexact = max(inexact, np.abs(v[again != v]).max(initial=0))
    assert 2.0 ** -14 < inexact / largest < 2.0 ** -13.8


def test_exponents(host):
    """The least power of two that takes a magnitude to at most 448, at its borders and at the range's ends."""
    f = np.array([448.0, np.nextafter(np.float32(448), np.float32(1e9)), 1.0, 1.75, 1.7500001, 3.5, 3.6, 0.0, 1e-45,
                  2.0 ** -32 * 448, 2.0 ** -32 * 449, 2.0 ** 31 * 448, 2.0 ** 31 * 449, 3.4e38, 2.0 ** -126], np.float32)
    for top in np.concatenate([f, np.exp(np.random.default_rng(0).uniform(-60, 60, 2000)).astype(np.float32)]):
        e = host.exponent(int(top.view(np.uint32)))
        assert e == mo.exponent(float(top)), top
        if -32 < e < 31:
            assert float(top) <= 448 * 2.0 ** e and float(top) > 224 * 2.0 ** e
    for e in range(-32, 32):
        assert host.exponent_of(int(np.float32(2.0 ** e).view(np.uint32))) == e
    for bits in (0, 0x7F800000, 0x7FC00000, 0xFFFFFFFF, 1):  # what is no scale stays in range
        assert -32 <= host.exponent_of(bits) <= 31


@pytest.mark.parametrize("d,page,hkv", [(32, 32, 1), (64, 64, 2), (96, 32, 3), (128, 256, 2)])
def test_locate_and_scales(d, page, hkv):
    desc = tlm.paged_desc(2 * hkv, hkv, d, 4 * page, page_tokens=page, kv_fmt=tlm.FMT_F8)
    size = mo.page_bytes(hkv, page, d)
    assert tlm.paged_page_bytes(desc) == size and size % 128 == 0
    table = [2, 0, 5]
    positions = np.concatenate([np.arange(page), [page, 2 * page - 1, 3 * page - 1]])
    want_k = mo.places8(table, positions, hkv, page, d, mo.k8_at)
    want_v = mo.places8(table, positions, hkv, page, d, mo.v8_at)
    want_s = mo.scales_at(table, positions, hkv, page, d)
    for i in list(range(0, page, 7)) + [page, page + 1, page + 2]:
        for h in range(hkv):
            assert tlm.paged_scale_at(desc, 6, table, int(positions[i]), h) == 4 * want_s[i, h]
            for c in range(0, d, 5):
                assert tlm.paged_locate(desc, 6, table, int(positions[i]), h, c) == (want_k[i, h, c], want_v[i, h, c])
    codes = set(range(2 * size, 2 * size + hkv * page * d))
    assert set(want_k[:page].ravel()) == codes and set(want_v[:page].ravel()) == codes
    at = set(want_s[:page].ravel() * 4)
    assert len(at) == hkv * page // 32 and min(at) == 2 * size + hkv * page * d and max(at) + 4 <= 3 * size


def test_layout_functions(host):
    t, c = np.meshgrid(np.arange(64), np.arange(96), indexing="ij")
    for tok, dim in ((0, 0), (17, 33), (31, 95), (32, 8), (63, 64), (40, 31)):
        assert host.k_at(tok, dim, 96) == mo.k8_at(tok, dim, 96) and host.v_at(tok, dim, 96) == mo.v8_at(tok, dim, 96)
    assert np.unique(mo.k8_at(t, c, 96)).size == t.size and np.unique(mo.v8_at(t, c, 96)).size == t.size


def test_locate_past_32_bits():
    desc = tlm.paged_desc(32, 8, 128, 1 << 20, page_tokens=256, kv_fmt=tlm.FMT_F8)
    size = tlm.paged_page_bytes(desc)
    k, v = tlm.paged_locate(desc, 1 << 20, [(1 << 20) - 1], 255, 7, 127)
    assert k == v == ((1 << 20) - 1) * size + 8 * 256 * 128 - 1 > 1 << 37
    assert tlm.paged_scale_at(desc, 1 << 20, [(1 << 20) - 1], 255, 7) == ((1 << 20) - 1) * size + 8 * 256 * 128 + 63 * 4


@pytest.mark.parametrize("shift", [5, 6, 10])
def test_pages_in_use(host, shift):
    rng = np.random.default_rng(shift)
    page = 1 << shift
    cases = [(0, 0, 0, 0), (0, 1, 0, 0), (0, 0, 5, 7), (31, 2, 1, 0), (100, 1, 1, 1), (100, 400, 50, 200), (5, 1, 100, 300)]
    cases += [tuple(int(x) for x in np.exp(rng.uniform(0, 8, 4)).astype(int) - 1) for _ in range(500)]
    for start, rows, window, sinks in cases:
        out = (ctypes.c_int * 3)()
        host.use(start, rows, window, sinks, shift, out)
        a, b, e = out
        assert 0 <= a <= b <= e
        got = list(range(a)) + list(range(b, e))
        assert got == mo.pages_in_use(start, rows, window, sinks, page), (start, rows, window, sinks)
    host.use(1 << 30, 1 << 22, 1 << 30, 1 << 30, shift, out)  # no overflow
    assert list(out) == [0, 0, ((1 << 30) + (1 << 22)) >> shift]
    host.use(1 << 30, 1, 3, 1 << 30, shift, out)
    assert out[0] == out[1] == ((1 << 30) - 2) >> shift


def test_shapes_refused():
    for fmt in (0, 2, 5, -1):
        desc = tlm.paged_desc(4, 2, 64, 100, page_tokens=32, kv_fmt=fmt)
        refused(tlm.TLM_ERR_INVALID, tlm.paged_page_bytes, desc)
    desc = tlm.paged_desc(4, 2, 64, 100, page_tokens=32, kv_fmt=tlm.FMT_F16)
    assert tlm.paged_page_bytes(desc) == 2 * 32 * 64 * 2
    refused(tlm.TLM_ERR_INVALID, tlm.paged_scale_at, desc, 4, [0, 1], 0, 0)  # it has no scales
    desc = tlm.paged_desc(4, 2, 64, 100, page_tokens=32, kv_fmt=tlm.FMT_F8)
    for position in (-1, 100, 64):
        refused(tlm.TLM_ERR_RANGE, tlm.paged_scale_at, desc, 4, [0, 1], position, 0)
    for head in (-1, 2):
        refused(tlm.TLM_ERR_INVALID, tlm.paged_scale_at, desc, 4, [0, 1], 0, head)
    refused(tlm.TLM_ERR_RANGE, tlm.paged_scale_at, desc, 4, [0, 4], 32, 0)


def test_null_arguments_refused():
    L, r, g = tlm.lib(), tlm.PagedRequest(), tlm.LogitRules()
    for rc in (L.tlm_paged_set_sinks(None, 1), L.tlm_paged_page_bytes(None, None), L.tlm_op_paged_reserve(None, r),
               L.tlm_paged_scale_at(None, 1, None, 1, 0, 0, None), L.tlm_op_adjust_logits(None, g),
               L.tlm_op_adjust_logits(None, None)):
        assert rc == tlm.TLM_ERR_INVALID
        assert L.tlm_last_error().startswith((b"TLMPaged: ", b"TLMLogitRules: "))


def test_histories_longer_than_a_sequence_are_refused():
    """A sequence has at most 2^30 positions; indexes into a longer history would pass 31 bits."""
    some = (ctypes.c_uint8 * 4096)()  # a context that the refusal does not look at, and buffers that nothing reads
    at = ctypes.addressof(some)
    for width in ((1 << 30) + 1, (1 << 31) - 4096, (1 << 31) - 1):
        r = tlm.LogitRules(logits=at, out=at, history=1 << 40, seqs=1, tokens=1, vocab=10, history_width=width)
        assert tlm.lib().tlm_op_adjust_logits(at, r) == tlm.TLM_ERR_INVALID
        assert tlm.lib().tlm_last_error() == b"TLMLogitRules: a history of %d, at most %d" % (width, 1 << 30)


def test_buffers_that_are_too_small_are_refused():
    """A byte too few is refused when the arguments are put together."""
    p = tlm.Paged.__new__(tlm.Paged)
    p.ctx, p.ptr, p.desc = None, None, tlm.paged_desc(6, 2, 64, 100, page_tokens=32, kv_fmt=tlm.FMT_F8)
    p.sizes = tlm.paged_sizes(p.desc)
    assert p.page_bytes() == 2 * 32 * 64 + 128
    small = buffer(1 << 10)
    says("k_pages holds", p.batch, buffer(3 * p.page_bytes() - 1), buffer(3 * p.page_bytes()), 3, small, 4, small, 5, 7)
    need = dict(lengths=20, tables=80, refs=12, starts=20, counts=20, slots=8 * 35, out_tables=80, out_refs=12)

    def request(**sizes):
        b = {k: buffer(n) for k, n in {**need, **sizes}.items()}
        return p.request(b["lengths"], b["tables"], 4, b["refs"], 3, b["starts"], 5, 7, counts=b["counts"],
                         slots=b["slots"], out_tables=b["out_tables"], out_refs=b["out_refs"])

    says("null", p.reserve, request())
    for name, n in need.items():
        says(f"{name} holds", request, **{name: n - 1})

    s, t, v, h, nb = 3, 4, 100, 9, 5
    need = dict(logits=4 * s * t * v, out=4 * s * t * v, counts=4 * s, history=4 * s * h, history_counts=4 * s,
                drafts=4 * s * (t - 1), repetition=4 * s, frequency=4 * s, presence=4 * s, bias_ids=4 * s * nb,
                biases=4 * s * nb, masks=4 * s * t * 4)

    class Ctx:
        ptr = None

    def rules(**sizes):
        b = {k: buffer(n) for k, n in {**need, **sizes}.items()}
        return tlm.logit_rules(b.pop("logits"), s, t, v, history_width=h, bias_width=nb, **b)

    says("invalid argument", tlm.adjust_logits, Ctx, rules())
    for name, n in need.items():
        says(f"{name} holds", rules, **{name: n - 1})


def test_plain_reservation_keeps_count():
    """What the tables hold and what the counts say agree after steps of every kind."""
    rng = np.random.default_rng(1)
    n, width, page, pages = 9, 12, 32, 60
    for window, sinks in ((0, 0), (70, 0), (70, 40), (1, 200)):
        tables, refs = np.full((n, width), -1, np.int32), np.zeros(pages, np.int32)
        refs[rng.permutation(pages)[:7]] = 1  # others'
        others, lengths = refs.copy(), np.zeros(n, np.int64)
        for _ in range(60):
            counts = rng.integers(0, 40, n)
            tables, refs, starts, slots, bad, lost = mo.reserve(tables, refs, lengths, counts, 40, window, sinks, page, 9999)
            assert not lost
            held = np.bincount(tables[tables >= 0], minlength=pages)
            assert np.array_equal(held + others, refs) and held.max() <= 1
            taken = slots[slots >= 0]
            assert np.unique(taken).size == taken.size
            for s in range(n):
                said = int((slots[s] >= 0).sum())
                assert (starts[s] >= 0) == (said > 0)
                if starts[s] >= 0:
                    lengths[s] += rng.integers(0, said + 1)
            for s in range(n):
                if lengths[s] > 300 or rng.random() < 0.05:
                    lengths[s] = -1
                elif lengths[s] < 0:
                    lengths[s] = 0
