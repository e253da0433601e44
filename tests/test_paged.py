"""The paged caches' index arithmetic and the refusals, on the host: the layout as a
bijection, rows and pages that are out of range, and what the entry points refuse
before any device is touched."""
import ctypes
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from test_host import header_struct_fields
import paged_oracle as po
import three_llm_amd.tlm as tlm

SHIM = """
#include "tlm_paged.h"
using namespace tlm;
extern "C" int rows(int start, int count, int tokens, int limit, int* bad) {
  bool b;
  const int r = paged_rows(start, count, tokens, limit, &b);
  *bad = b;
  return r;
}
extern "C" int page(const int32_t* t, int p, int shift, int n) { return paged_page(t, p, shift, n); }
extern "C" int limit(int m, int w, int s) { return paged_limit(m, w, s); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """The kernels' own bounds arithmetic, built for the host."""
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", str(ROOT / "three-llm_amd" / "csrc"), "-o",
                    str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("cname,pytype", [("tlm_paged_desc", tlm.PagedDesc), ("tlm_paged_batch", tlm.PagedBatch)])
def test_structs_match_the_header(cname, pytype):
    assert [f for f, _ in pytype._fields_] == header_struct_fields(cname)


@pytest.mark.parametrize("start,count,tokens,limit,want,bad", [
    (0, 1, 1, 1, 1, 0), (-1, 1, 1, 8, 0, 0), (-2 ** 31, 1, 1, 8, 0, 0), (3, 0, 4, 8, 0, 0), (3, -2 ** 31, 4, 8, 0, 0),
    (4, 4, 4, 8, 4, 0), (5, 4, 4, 8, 3, 1), (8, 1, 4, 8, 0, 1), (2 ** 31 - 1, 2 ** 31 - 1, 16, 8, 0, 1),
    (0, 9, 4, 64, 4, 1), (2 ** 31 - 2, 16, 16, 2 ** 31 - 1, 1, 1)])
def test_rows_that_are_there(host, start, count, tokens, limit, want, bad):
    b = ctypes.c_int()
    assert host.rows(start, count, tokens, limit, ctypes.byref(b)) == want
    assert b.value == bad


def test_pages_out_of_the_pool(host):
    t = np.array([3, -1, 4, 0, 2 ** 31 - 1, -2 ** 31], np.int32)
    got = [host.page(t.ctypes.data_as(ctypes.c_void_p), 32 * i + 31, 5, 4) for i in range(t.size)]
    assert got == [3, -1, -1, 0, -1, -1]
    assert host.limit(100, 2, 5) == 64 and host.limit(50, 2, 5) == 50
    assert host.limit(2 ** 30, 2 ** 31 - 1, 10) == 2 ** 30  # the product passes 32 bits


@pytest.mark.parametrize("fmt,e", [(tlm.FMT_F16, 8), (tlm.FMT_F32, 4)])
@pytest.mark.parametrize("d,page,hkv", [(32, 32, 1), (64, 64, 2), (96, 32, 3), (128, 128, 2)])
def test_locate_is_a_bijection_in_the_documented_order(fmt, e, d, page, hkv):
    desc = tlm.paged_desc(2 * hkv, hkv, d, 4 * page, page_tokens=page, kv_fmt=fmt)
    table = [2, 0, 5]
    seen_k, seen_v = set(), set()
    positions = list(range(page)) + [page, 2 * page - 1, 3 * page - 1]
    want_k = po.places(table, positions, hkv, page, d, e, po.k_at)
    want_v = po.places(table, positions, hkv, page, d, e, po.v_at)
    step = max(1, d // 32)
    for i, p in enumerate(positions):
        for h in range(hkv):
            for c in range(0, d, step):
                k, v = tlm.paged_locate(desc, 6, table, p, h, c)
                assert (k, v) == (want_k[i, h, c], want_v[i, h, c])
    seen_k, seen_v = set(want_k[:page].ravel()), set(want_v[:page].ravel())
    whole = set(range(2 * hkv * page * d, 3 * hkv * page * d))
    assert seen_k == whole and seen_v == whole


def test_locate_past_32_bits():
    desc = tlm.paged_desc(32, 8, 128, 1 << 20, page_tokens=256)
    k, v = tlm.paged_locate(desc, 1 << 20, [(1 << 20) - 1], 255, 7, 127)
    assert k == v == (1 << 20) * 8 * 256 * 128 - 1


def refused(code, call, *args, **kw):
    with pytest.raises(tlm.TlmError) as e:
        call(*args, **kw)
    assert e.value.code == code and ":" in str(e.value)


@pytest.mark.parametrize("change", [
    dict(heads=0), dict(heads=3), dict(heads=34), dict(heads=2050, kv_heads=1025), dict(head_dim=48),
    dict(head_dim=256), dict(page_tokens=16), dict(page_tokens=48), dict(page_tokens=2048), dict(max_tokens=0),
    dict(max_tokens=2 ** 30 + 1), dict(kv_fmt=tlm.FMT_Q4), dict(sliding_window=-1), dict(rotary_dim=7),
    dict(rotary_dim=66)])
def test_shapes_refused(change):
    shape = dict(heads=4, kv_heads=2, head_dim=64, max_tokens=100, page_tokens=32,
                 inv_freq=np.ones(64, np.float32), rotary_dim=64)
    shape.update(change)
    desc = tlm.paged_desc(**shape)
    refused(tlm.TLM_ERR_INVALID, tlm.paged_locate, desc, 4, [0, 1, 2, 3], 0, 0, 0)


def test_places_refused():
    desc = tlm.paged_desc(4, 2, 64, 100, page_tokens=32)
    for position in (-1, 100, 64, 2 ** 31 - 1):  # the table holds 64, the model 100
        refused(tlm.TLM_ERR_RANGE, tlm.paged_locate, desc, 4, [0, 1], position, 0, 0)
    for entry in (-1, 4, 2 ** 31 - 1, -2 ** 31):
        refused(tlm.TLM_ERR_RANGE, tlm.paged_locate, desc, 4, [0, entry], 32, 0, 0)
    for head, dim in ((2, 0), (-1, 0), (0, 64), (0, -1)):
        refused(tlm.TLM_ERR_INVALID, tlm.paged_locate, desc, 4, [0, 1], 0, head, dim)
    desc.inv_freq = None
    desc.rotary_dim = 64
    refused(tlm.TLM_ERR_INVALID, tlm.paged_locate, desc, 4, [0, 1], 0, 0, 0)


def test_null_arguments_refused():
    L, b = tlm.lib(), tlm.PagedBatch()
    for rc in (L.tlm_paged_create(None, None, None), L.tlm_op_paged_append(None, ctypes.byref(b), None, None),
               L.tlm_op_paged_attention(None, ctypes.byref(b), None, tlm.FMT_F16, None), L.tlm_paged_status(None),
               L.tlm_op_verify_drafts(None, None, None, None, None, None, 1, 1, 8, 1.0, None, None)):
        assert rc == tlm.TLM_ERR_INVALID
        assert L.tlm_last_error().startswith((b"TLMPaged: ", b"TLMVerify: "))
    L.tlm_paged_destroy(None)


def buffer(nbytes):
    b = tlm.Buffer.__new__(tlm.Buffer)  # an address that no call gets as far as
    b.ctx, b.nbytes, b.ptr = None, nbytes, ctypes.c_void_p(4096)
    return b


def says(part, call, *args, **kw):
    with pytest.raises(tlm.TlmError) as e:
        call(*args, **kw)
    assert e.value.code == tlm.TLM_ERR_INVALID and part in str(e.value), str(e.value)


@pytest.mark.parametrize("fmt,size", [(tlm.FMT_F16, 2), (tlm.FMT_F32, 4)])
def test_rows_that_a_buffer_does_not_hold_are_refused(fmt, size):
    """A byte too few is refused before the call; enough reaches it, and it has no handle here."""
    p = tlm.Paged.__new__(tlm.Paged)
    p.ctx, p.ptr, p.desc = None, None, tlm.paged_desc(6, 2, 64, 100, page_tokens=32)
    p.sizes = tlm.paged_sizes(p.desc)
    pool, small = buffer(3 * p.page_bytes()), buffer(1 << 10)
    b = p.batch(pool, pool, 3, small, 4, small, 5, 7)
    rows, whole = 35, buffer(35 * 10 * 64 * 4)
    qkv, q, out = rows * 10 * 64 * 4, rows * 6 * 64 * 4, rows * 6 * 64 * size
    says("qkv holds", p.append, b, buffer(qkv - 1), whole)
    says("q holds", p.append, b, whole, buffer(q - 1))
    says("q holds", p.attention, b, buffer(q - 1), whole, fmt)
    says("out holds", p.attention, b, whole, buffer(out - 1), fmt)
    says("null", p.append, b, buffer(qkv), buffer(q))
    says("null", p.append, b, buffer(qkv))
    says("null", p.attention, b, buffer(q), buffer(out), fmt)
    # a batch of another handle, whose pages are smaller
    p.sizes = tlm.paged_sizes(tlm.paged_desc(6, 2, 64, 100, page_tokens=64))
    says("k_pages holds", p.append, b, whole, whole)
    says("k_pages holds", p.attention, b, whole, whole, fmt)


def test_verification_buffers_that_are_too_small_are_refused():
    s, t, v = 3, 4, 100
    need = dict(logits_buf=4 * s * t * v, accepted=4 * s, out_tokens=4 * s * t, drafts=4 * s * (t - 1),
                draft_logits=4 * s * (t - 1) * v, counts=4 * s, uniforms=4 * s * t)

    class Ctx:
        ptr = None

    def call(temperature, **sizes):
        b = {k: buffer(n) for k, n in {**need, **sizes}.items()}
        tlm.verify_drafts(Ctx, b.pop("logits_buf"), s, t, v, b.pop("accepted"), b.pop("out_tokens"),
                          temperature=temperature, **b)

    for temperature in (0.0, 0.7):
        says("invalid argument", call, temperature)
        for name, n in need.items():
            read = temperature > 0 or name not in ("draft_logits", "uniforms")
            says("holds" if read else "invalid argument", call, temperature, **{name: n - 1})
