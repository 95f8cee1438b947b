"""Refusals of the paged-cache operators: every bad argument is an error code with a message, before
any device work (pointers here are never followed)."""
from __future__ import annotations

import ctypes as C

import pytest

P = 1 << 20   # a 16- and 256-byte aligned address


def pool(pkg, **kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, n_pages=4, page_size=16, kv_heads=2, head_dim=64, format=1)
    f.update(kw)
    return C.byref(pkg._abi.PagePool(**f))


def store(pkg, lib, pl=None, **kw):
    a = dict(k=P, v=P, type=0, ks=128, vs=128, tokens=1, slots=P)
    a.update(kw)
    return lib.g4_op_page_store(pl or pool(pkg), a["k"], a["v"], a["type"], a["ks"], a["vs"], a["tokens"], a["slots"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(k=None), "null"), (dict(format=3), "format"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=2048), "page_size"), (dict(n_pages=0), "pages"),
    (dict(kv_heads=0), "heads"), (dict(n_pages=1 << 28), "pages"), (dict(k_scale=None), "scales"), (dict(v=P + 8), "aligned"),
])
def test_pool_refused(pkg, lib, bad, text):
    for rc in (store(pkg, lib, pool(pkg, **bad)),
               lib.g4_op_page_read(pool(pkg, **bad), P, 1, 0, P, P, 128, 128, None),
               lib.g4_op_paged_attention_workspace(pool(pkg, **bad), 0, 8, 1, 1, 1, 1, 0, C.byref(C.c_uint64()))):
        assert rc in (-1, -5)
        assert text in pkg._abi.last_error()


@pytest.mark.parametrize("bad,text", [
    (dict(k=None), "null"), (dict(slots=None), "null"), (dict(type=2), "type"), (dict(tokens=-1), "tokens"),
    (dict(ks=130), "aligned"), (dict(v=P + 4), "aligned"), (dict(ks=64), "apart"), (dict(type=1, ks=132), "aligned"),
])
def test_store_refused(pkg, lib, bad, text):
    assert store(pkg, lib, **bad) == -1
    assert text in pkg._abi.last_error()


def test_nothing_to_do_is_no_error(pkg, lib):
    assert store(pkg, lib, tokens=0) == 0
    assert lib.g4_op_page_read(pool(pkg), P, 0, 0, P, P, 128, 128, None) == 0
    assert attention(pkg, lib, rows=0) == 0 and attention(pkg, lib, batch=0) == 0
    assert drafts(pkg, lib, batch=0) == 0


def attention(pkg, lib, pl=None, **kw):
    a = dict(q=P, qs=512, out=P, os=512, lse=None, type=0, heads=8, rows=3, batch=2, begin=P, pos=P, kv=P, table=P, ts=4,
             max_q=2, max_kv=64, window=0, scale=1.0, ws=P, wb=1 << 40)
    a.update(kw)
    return lib.g4_op_paged_attention(pl or pool(pkg), a["q"], a["qs"], a["out"], a["os"], a["lse"], a["type"], a["heads"],
                                     a["rows"], a["batch"], a["begin"], a["pos"], a["kv"], a["table"], a["ts"], a["max_q"],
                                     a["max_kv"], a["window"], a["scale"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(q=None), "null"), (dict(table=None), "null"), (dict(ws=None), "null"), (dict(type=5), "type"), (dict(heads=7), "heads"),
    (dict(heads=0), "heads"), (dict(heads=258), "heads"), (dict(rows=-1), "rows"), (dict(batch=70000), "batch"),
    (dict(max_q=-1), "max_q"), (dict(max_kv=65), "page tables"), (dict(window=-1), "window"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(qs=514), "aligned"), (dict(os=256), "apart"), (dict(wb=1000), "workspace"),
    (dict(ws=P + 16), "workspace"),
])
def test_attention_refused(pkg, lib, bad, text):
    assert attention(pkg, lib, **bad) in (-1, -5)
    assert text in pkg._abi.last_error()


def drafts(pkg, lib, **kw):
    a = dict(logits=P, ld=100, type=0, vocab=100, rows=4, batch=2, begin=P, drafts=P, probs=None, lp=0, u=P, gumbel=P, lg=100,
             temp=P, most=3, tokens=P, logprobs=P, counts=P, ws=P, wb=1 << 40)
    a.update(kw)
    return lib.g4_op_verify_drafts(a["logits"], a["ld"], a["type"], a["vocab"], a["rows"], a["batch"], a["begin"], a["drafts"],
                                   a["probs"], a["lp"], a["u"], a["gumbel"], a["lg"], a["temp"], a["most"], a["tokens"],
                                   a["logprobs"], a["counts"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("bad,text", [
    (dict(logits=None), "null"), (dict(gumbel=None), "null"), (dict(counts=None), "null"), (dict(type=3), "type"),
    (dict(vocab=0), "vocab"), (dict(rows=-1), "rows"), (dict(batch=65536), "batch"), (dict(most=-1), "max_drafts"),
    (dict(most=256), "max_drafts"), (dict(ld=99), "apart"), (dict(lg=99), "apart"), (dict(probs=P, lp=99), "apart"),
    (dict(logits=P + 2), "aligned"), (dict(gumbel=P + 2), "aligned"), (dict(wb=100), "workspace"), (dict(ws=P + 8), "workspace"),
])
def test_drafts_refused(pkg, lib, bad, text):
    assert drafts(pkg, lib, **bad) in (-1, -5)
    assert text in pkg._abi.last_error()


def test_workspace_sizes(pkg, lib):
    n = C.c_uint64()
    assert lib.g4_op_paged_attention_workspace(pool(pkg), 0, 8, 3, 2, 2, 64, 0, C.byref(n)) == 0 and n.value >= 65536 * 4
    assert lib.g4_op_verify_drafts_workspace(100, 4, 2, 3, C.byref(n)) == 0 and n.value > 65536 * 4
    assert lib.g4_op_paged_attention_workspace(pool(pkg), 0, 8, 3, 2, 2, 64, 0, None) == -1
    assert lib.g4_op_verify_drafts_workspace(0, 4, 2, 3, C.byref(n)) == -1


def test_errors_entry_refuses_null(pkg, lib):
    assert lib.g4_op_paged_errors(None) == -1
