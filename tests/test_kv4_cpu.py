"""Refusals of the 4-bit cache and scoring entry points: every bad argument
comes back as MG_ERR_ARG with a message, before any device call (so this runs
without a GPU; the pointers are never followed)."""
import ctypes as C

import numpy as np
import pytest

from midge_b200 import abi
from tests import kv4_ref as ref

P = 4096  # a pointer that is never read here


def cache(**kw):
    f = dict(n_kv_heads=8, head_dim=64, page_size=64, n_seqs=2, n_pages=16, pages=P, table=P, ld_table=8)
    return abi.MgKv4(**{**f, **kw})


BAD_CACHE = [dict(head_dim=96), dict(head_dim=0), dict(page_size=16), dict(page_size=48), dict(page_size=8192),
             dict(n_kv_heads=0), dict(n_pages=0), dict(n_seqs=0), dict(ld_table=0), dict(ld_table=1 << 40),
             dict(pages=None), dict(table=None), dict(pages=P + 8), dict(n_pages=1 << 31)]


def refused(rc, word=b""):
    assert rc == abi.MG_ERR_ARG
    assert word in abi.lib.mg_last_error()


def append(c, act=0, n=1, heads=64, q=P, ldq=4096, k=P, ldk=512, v=P, ldv=512, eps=1e-6, co=P, si=P, rows=8, pos=P,
           qo=P, ldo=4096):
    return abi.lib.mg_kv4_append(c, act, n, heads, q, ldq, k, ldk, v, ldv, None, None, eps, co, si, rows, None, pos,
                                 qo, ldo, None)


def attn(c, act=0, heads=64, q=P, ldq=4096, qs=P, kl=P, mq=1, mk=64, win=0, out=P, ldo=4096, work=P, nwork=1 << 40):
    return abi.lib.mg_kv4_attn(c, act, heads, q, ldq, qs, kl, mq, mk, 0.125, win, None, out, ldo, work, nwork, None)


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_cache_refused_everywhere(kw):
    c = C.byref(cache(**kw))
    refused(append(c), b"kv4")
    refused(attn(c), b"kv4")
    refused(abi.lib.mg_kv4_read(c, 0, 1, None, P, P, 512, P, 512, None), b"kv4")
    refused(abi.lib.mg_kv4_attn_work(c, 64, 1, 64), b"kv4")
    refused(append(None), b"null")


@pytest.mark.parametrize("kw", [dict(act=3), dict(act=-1), dict(n=-1), dict(heads=-1), dict(q=None), dict(ldq=4095),
                                dict(k=None), dict(v=None), dict(ldk=511), dict(ldv=511), dict(co=None),
                                dict(si=None), dict(rows=0), dict(pos=None), dict(qo=None), dict(ldo=100),
                                dict(eps=-1.0)])
def test_append_refusals(kw):
    refused(append(C.byref(cache()), **kw), b"kv4_append")


def test_read_refusals():
    c = C.byref(cache())
    for act, n, pos, k, ldk, v, ldv in [(5, 1, P, P, 512, P, 512), (0, -1, P, P, 512, P, 512),
                                        (0, 1, None, P, 512, P, 512), (0, 1, P, None, 0, None, 0),
                                        (0, 1, P, P, 511, P, 512), (0, 1, P, P, 512, P, 0)]:
        refused(abi.lib.mg_kv4_read(c, act, n, None, pos, k, ldk, v, ldv, None), b"kv4_read")


@pytest.mark.parametrize("kw", [dict(act=3), dict(heads=0), dict(heads=60), dict(heads=8 * 65), dict(q=None),
                                dict(ldq=4095), dict(qs=None), dict(kl=None), dict(mq=0), dict(mq=1 << 20),
                                dict(mk=-1), dict(win=-1), dict(out=None), dict(ldo=4095)])
def test_attn_refusals(kw):
    refused(attn(C.byref(cache()), **kw), b"kv4_attn")


def test_attn_workspace_too_small():
    c = C.byref(cache())
    need = abi.check_size(abi.lib.mg_kv4_attn_work(c, 64, 1, 512))
    if need:
        refused(attn(c, mk=512, nwork=need - 1), b"workspace")
        refused(attn(c, mk=512, work=None), b"workspace")


def test_logprobs_refusals():
    ok = dict(act=0, x=P, ld=100, V=100, n=2, ids=P, n_ids=1, top=5, lp=P, ent=P, ai=P, al=P)
    for kw in [dict(act=7), dict(x=None), dict(ld=99), dict(V=0), dict(n=-1), dict(ids=None), dict(lp=None),
               dict(n_ids=-1), dict(top=33), dict(top=-1), dict(ent=None), dict(ai=None), dict(al=None),
               dict(V=1 << 31, ld=1 << 31)]:
        a = {**ok, **kw}
        refused(abi.lib.mg_logprobs(a["act"], a["x"], a["ld"], a["V"], a["n"], a["ids"], a["n_ids"], a["top"], a["lp"],
                                    a["ent"], a["ai"], a["al"], P, 1 << 40, None), b"logprobs")
    assert abi.lib.mg_logprobs_work(0, 1, 1) == abi.MG_ERR_ARG


def test_nothing_to_do_is_ok():
    assert append(C.byref(cache()), n=0) == abi.MG_OK
    assert abi.lib.mg_kv4_read(C.byref(cache()), 0, 0, None, P, P, 512, None, 0, None) == abi.MG_OK
    assert abi.lib.mg_logprobs(0, P, 100, 100, 0, None, 0, 0, None, P, None, None, P, 1 << 40, None) == abi.MG_OK


def test_page_bytes():
    assert abi.lib.mg_kv4_page_bytes(8, 64, 64) == 8 * 2 * 34 * 64
    assert abi.lib.mg_kv4_page_bytes(4, 128, 32) == 4 * 34 * 128
    assert abi.lib.mg_kv4_page_bytes(8, 80, 64) == abi.MG_ERR_ARG
    with pytest.raises(abi.MidgeError):
        abi.check_size(abi.lib.mg_kv4_page_bytes(8, 64, 33))


@pytest.mark.parametrize("D", [64, 128])
def test_tile_places_are_a_permutation(D):
    """Every byte of a tile belongs to exactly one pair of codes or one scale."""
    p, d, g = np.arange(32)[:, None], np.arange(0, D, 2)[None], np.arange(D // 32)[None]
    at = np.concatenate([x.ravel() for x in (ref.k_place(p, d, D), ref.v_place(p, d, D), ref.k_scale_place(p, g, D),
                                             ref.v_scale_place(p, g, D))])
    assert sorted(at) == list(range(34 * D))
    assert np.array_equal(ref.k_place(p, d, D), ref.k_place(p, d + 1, D))


def test_quantiser_of_the_oracle():
    """Its codes are the nearest (64-bit search over all sixteen) with ties to
    even, its scale the least that keeps the largest magnitude in range."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)) * np.exp(rng.uniform(-8, 8, (50, 1)))
    c, sb = ref.quantise(x)
    v = ref.values(c, sb)
    s = np.repeat(ref.e5m2(sb), 32, -1)
    allv = np.concatenate([ref.MAG, -ref.MAG])
    best = np.abs(x[..., None] - s[..., None] * allv).min(-1)
    assert np.allclose(np.abs(x - v), best, rtol=1e-12, atol=0)
    top = np.abs(x.reshape(50, 2, 32)).max(-1)
    assert (ref.e5m2(sb) * 6 >= top).all() and (ref.e5m2(sb - 1) * 6 < top).all()
    t = np.zeros((1, 32))
    t[0, :8] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5]
    assert list(ref.quantise(t)[0][0, :8]) == [7, 0, 2, 2, 4, 4, 6, 6]
