"""Refusals of the attention block's entry points: argument checks on the host, before any device work."""
import ctypes

import pytest

import conftest

OK, INVAL = 0, 1
P, Q = 0x100000, 0x200000  # stand-ins for device addresses: no refused call reaches the device


@pytest.fixture(scope="module")
def L():
    return conftest.load_amd().lib()


def view(data=P, heads=2, token=256, head=128):
    return conftest.load_amd().HeadView(data, heads, token, head)


def call_rope(L, q=None, k=None, qo=None, ko=None, **kw):
    a = dict(xt=1, tokens=3, d=128, qw=None, kw=None, eps=1e-6, pos=P, freq=P, rot=128, pairs=0, scale=1.0, yt=1)
    a.update(kw)
    ref = lambda v: None if v is None else ctypes.byref(v)  # noqa: E731
    return L.exl3_hip_qk_norm_rope(ref(q or view()), ref(k), a["xt"], a["tokens"], a["d"], a["qw"], a["kw"], a["eps"],
                                   a["pos"], a["freq"], a["rot"], a["pairs"], a["scale"], ref(qo or view(Q)), ref(ko),
                                   a["yt"], None)


def test_rope_refusals(L):
    assert call_rope(L, tokens=0) == OK
    for bad in (dict(xt=2), dict(yt=-1), dict(d=4), dict(d=12), dict(d=264), dict(rot=8), dict(rot=144), dict(pos=None),
                dict(freq=None), dict(pos=P + 2), dict(qw=P + 1), dict(kw=P + 2), dict(eps=-1.0),
                dict(eps=float("nan")), dict(tokens=1 << 31)):
        assert call_rope(L, **bad) == INVAL, bad
    assert L.exl3_hip_qk_norm_rope(None, None, 1, 1, 128, None, None, 0.0, P, P, 128, 0, 1.0, ctypes.byref(view()), None,
                                   1, None) == INVAL
    for q in (view(None), view(P + 1), view(heads=0), view(heads=2000), view(token=1 << 41), view(heads=3)):
        assert call_rope(L, q=q) == INVAL  # the last: another head count than the output's
    for qo in (view(Q, head=64), view(Q, token=255), view(Q, token=100, head=300)):
        assert call_rope(L, qo=qo) == INVAL  # heads that overlap
    assert call_rope(L, qo=view(P, token=512)) == INVAL         # in place with other strides
    assert call_rope(L, qo=view(P), yt=0) == INVAL              # in place with another type
    assert call_rope(L, k=view(P, 1)) == INVAL                  # keys without an output
    assert call_rope(L, ko=view(P, 1)) == INVAL
    assert call_rope(L, k=view(P, 1), ko=view(Q, 2)) == INVAL


def test_page_bytes(L):
    f = L.exl3_hip_kv_page_bytes
    assert f(4, 8, 128, 256) == 8 * 256 * 2 * (64 + 8)
    assert f(8, 1, 64, 16) == 16 * 2 * (64 + 4)
    for bad in ((3, 8, 128, 256), (4, 0, 128, 256), (4, 1025, 128, 256), (4, 8, 96, 256), (4, 8, 128, 0),
                (4, 8, 128, 8), (4, 8, 128, 24), (4, 8, 128, 65552)):
        assert f(*bad) == 0, bad


def call_write(L, k=None, v=None, **kw):
    a = dict(pages=P, count=4, bits=4, p=16, d=128, xt=1, tokens=3, slots=P, bad=None)
    a.update(kw)
    return L.exl3_hip_kv_cache_write(a["pages"], a["count"], a["bits"], a["p"], a["d"], ctypes.byref(k or view()),
                                     ctypes.byref(v or view()), a["xt"], a["tokens"], a["slots"], a["bad"], None)


def call_read(L, k=None, v=None, **kw):
    a = dict(pages=P, count=4, bits=4, p=16, d=128, yt=1, tokens=3, slots=P, bad=None)
    a.update(kw)
    return L.exl3_hip_kv_cache_read(a["pages"], a["count"], a["bits"], a["p"], a["d"], a["slots"], a["tokens"],
                                    ctypes.byref(k or view(Q)), ctypes.byref(v or view(2 * Q)), a["yt"], a["bad"], None)


def test_kv_cache_refusals(L):
    for call, t in ((call_write, "xt"), (call_read, "yt")):
        assert call(L, tokens=0) == OK
        for bad in (dict(pages=None), dict(pages=P + 8), dict(bits=5), dict(p=20), dict(d=96), dict(slots=None),
                    dict(slots=P + 4), dict(bad=P + 2), {t: 7}, dict(tokens=1 << 31), dict(count=1 << 31)):
            assert call(L, **bad) == INVAL, bad
        assert call(L, v=view(heads=1)) == INVAL
        assert call(L, k=view(None)) == INVAL
        assert call(L, k=view(P + 1)) == INVAL
    assert call_read(L, k=view(head=64)) == INVAL
    assert L.exl3_hip_kv_cache_write(P, 4, 4, 16, 128, None, ctypes.byref(view()), 1, 1, P, None, None) == INVAL
    assert L.exl3_hip_kv_cache_read(P, 4, 4, 16, 128, P, 1, ctypes.byref(view()), None, 1, None, None) == INVAL


def call_cached(L, q=None, out=None, **kw):
    a = dict(d=128, pages=P, count=4, bits=4, p=16, heads=1, table=P, stride=9, lens=P, seqs=2, q_len=1, ws=None, wb=0)
    a.update(kw)
    return L.exl3_hip_attention_cached(ctypes.byref(q or view()), ctypes.byref(out or view(Q)), a["d"], a["pages"],
                                       a["count"], a["bits"], a["p"], a["heads"], a["table"], a["stride"], a["lens"],
                                       a["seqs"], a["q_len"], 0.1, a["ws"], a["wb"], None)


def test_cached_refusals(L):
    assert call_cached(L, seqs=0) == OK
    for bad in (dict(d=80), dict(pages=None), dict(pages=P + 4), dict(count=0), dict(bits=2), dict(p=8), dict(heads=0),
                dict(heads=3), dict(heads=4), dict(table=None), dict(table=P + 1), dict(stride=0), dict(stride=1 << 30),
                dict(lens=None), dict(lens=P + 2), dict(seqs=65537), dict(q_len=0), dict(q_len=65537),
                dict(seqs=65536, q_len=65536), dict(ws=P + 16, wb=1 << 30)):
        assert call_cached(L, **bad) == INVAL, bad
    assert call_cached(L, out=view(P)) == INVAL
    assert call_cached(L, out=view(Q, heads=1)) == INVAL
    assert call_cached(L, out=view(Q, head=64)) == INVAL
    assert call_cached(L, q=view(heads=65, token=65 * 128), out=view(Q, heads=65, token=65 * 128)) == INVAL
    need = L.exl3_hip_attention_cached_workspace_bytes(2, 1, 128, 2, 1)
    assert need > 0 and call_cached(L, ws=P, wb=need - 1) == 3
    for bad in ((2, 0, 128, 2, 1), (3, 2, 128, 2, 1), (2, 1, 96, 2, 1), (2, 1, 128, 65537, 1), (2, 1, 128, 2, 0),
                (65, 1, 128, 1, 1)):
        assert L.exl3_hip_attention_cached_workspace_bytes(*bad) == 0, bad
    # a workspace serves every smaller call of the same heads
    sizes = [L.exl3_hip_attention_cached_workspace_bytes(32, 8, 128, s, 1) for s in (1, 2, 7, 64, 300)]
    assert sizes == sorted(sizes)


def call_prompt(L, q=None, k=None, v=None, out=None, **kw):
    a = dict(d=128, qs=P, ks=P, seqs=1, nq=3, nk=3, ws=None, wb=0)
    a.update(kw)
    return L.exl3_hip_attention_prompt(ctypes.byref(q or view()), ctypes.byref(k or view(heads=1)),
                                       ctypes.byref(v or view(heads=1)), ctypes.byref(out or view(Q)), a["d"], a["qs"],
                                       a["ks"], a["seqs"], a["nq"], a["nk"], 0.1, 1, a["ws"], a["wb"], None)


def test_prompt_refusals(L):
    assert call_prompt(L, seqs=0) == OK and call_prompt(L, nq=0) == OK
    for bad in (dict(d=32), dict(qs=None), dict(ks=None), dict(qs=P + 2), dict(seqs=65537), dict(nq=1 << 31),
                dict(nk=1 << 31)):
        assert call_prompt(L, **bad) == INVAL, bad
    assert call_prompt(L, k=view(heads=3), v=view(heads=3)) == INVAL
    assert call_prompt(L, v=view(heads=2)) == INVAL
    assert call_prompt(L, out=view(P)) == INVAL
    assert call_prompt(L, out=view(Q, heads=1)) == INVAL
    assert call_prompt(L, out=view(Q, token=200)) == INVAL
    assert call_prompt(L, q=view(P + 1)) == INVAL


def test_prompt_workspace(L):
    size = L.exl3_hip_attention_prompt_workspace_bytes
    need = size(2, 128, 1, 3, 4000)
    assert need > 0
    assert call_prompt(L, nk=4000, ws=P, wb=need - 1) == 3
    assert call_prompt(L, nk=4000, ws=P + 1, wb=need) == INVAL
    # none: short walks, workgroups enough, refused arguments
    for none in ((2, 128, 1, 3, 300), (32, 128, 1, 8192, 8192), (2, 128, 0, 3, 4000), (2, 128, 1, 0, 4000),
                 (2, 96, 1, 3, 4000), (0, 128, 1, 3, 4000)):
        assert size(*none) == 0, none
