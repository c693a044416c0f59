"""Refusals of the linear-attention block's entry points: argument checks on the host, before any device work."""
import ctypes

import pytest

import conftest

OK, INVAL, NO_SUPPORT = 0, 1, 2
P, Q, R, S = 0x100000, 0x200000, 0x300000, 0x400000  # stand-ins for device addresses: no refused call reaches the device
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def L():
    return conftest.load_amd().lib()


def view(data=P, heads=2, token=256, head=128):
    return conftest.load_amd().HeadView(data, heads, token, head)


def ref(v):
    return None if v is None else ctypes.byref(v)


def norm(L, x=None, gate=None, res=None, res_out=None, out=None, **kw):
    a = dict(xt=1, rt=0, tokens=3, width=128, weight=None, eps=1e-6, yt=1)
    a.update(kw)
    return L.exl3_hip_rms_norm(ref(x or view()), ref(gate), a["xt"], ref(res), ref(res_out), a["rt"], a["tokens"],
                               a["width"], a["weight"], a["eps"], ref(out or view(Q)), a["yt"], None)


def test_rms_norm(L):
    assert norm(L, tokens=0) == OK
    for bad in (dict(xt=2), dict(rt=-1), dict(yt=3), dict(width=0), dict(width=65537), dict(weight=P + 2), dict(eps=-1e-9),
                dict(eps=NAN), dict(eps=INF), dict(tokens=1 << 31)):
        assert norm(L, **bad) == INVAL, bad
    for x in (view(None), view(P + 1), view(heads=0), view(heads=1025), view(heads=3), view(token=1 << 41)):
        assert norm(L, x=x) == INVAL
    for out in (view(None), view(Q, heads=1), view(Q, head=64), view(Q, token=255)):
        assert norm(L, out=out) == INVAL
    assert norm(L, out=view(P, token=512)) == INVAL            # in place with other strides
    assert norm(L, out=view(P), yt=0) == INVAL                 # in place with another type
    assert norm(L, gate=view(Q)) == INVAL                      # out over the gate
    assert norm(L, gate=view(R, heads=1)) == INVAL
    assert norm(L, res=view(Q)) == INVAL                       # out over the residual
    assert norm(L, res=view(R, heads=1)) == INVAL
    assert norm(L, res_out=view(R)) == INVAL                   # no residual to keep the sum of
    assert norm(L, res=view(R), res_out=view(S, head=64)) == INVAL
    assert norm(L, res=view(R), res_out=view(R, token=512)) == INVAL
    for taken in (P, Q):                                       # the sum over x or over out
        assert norm(L, res=view(R), res_out=view(taken)) == INVAL
    assert norm(L, res=view(R), gate=view(S), res_out=view(S)) == INVAL


def conv(L, **kw):
    a = dict(x=P, xt=1, xs=64, tokens=6, channels=64, weight=P, width=4, bias=None, silu=1, starts=None, sequences=2,
             states=R, slots=4, sin=P, sout=P, y=Q, yt=1, ys=64)
    a.update(kw)
    return L.exl3_hip_short_conv(a["x"], a["xt"], a["xs"], a["tokens"], a["channels"], a["weight"], a["width"], a["bias"],
                                 a["silu"], a["starts"], a["sequences"], a["states"], a["slots"], a["sin"], a["sout"],
                                 a["y"], a["yt"], a["ys"], None)


PACKED_BAD = (dict(sequences=65537, starts=P), dict(tokens=(1 << 30) + 1, starts=P), dict(tokens=7), dict(starts=P + 2),
              dict(sin=P + 1), dict(sout=P + 2), dict(states=R + 8), dict(states=None), dict(states=None, sin=None),
              dict(slots=0), dict(slots=0, sout=None), dict(slots=(1 << 30) + 1))


def test_short_conv(L):
    assert conv(L, sequences=0, starts=P) == OK
    for bad in PACKED_BAD + (dict(xt=2), dict(yt=-1), dict(channels=0), dict(channels=(1 << 20) + 1), dict(width=1),
                             dict(width=5), dict(xs=63), dict(ys=63), dict(xs=1 << 41), dict(ys=1 << 41), dict(weight=None),
                             dict(weight=P + 1), dict(bias=P + 2), dict(x=P + 1), dict(y=Q + 1), dict(x=None), dict(y=None),
                             dict(y=P), dict(xs=1 << 40, tokens=1 << 10), dict(channels=1 << 20, xs=1 << 20, ys=1 << 20,
                                                                                slots=1 << 29)):
        assert conv(L, **bad) == INVAL, bad
    big = dict(starts=P, xs=1 << 18, ys=1 << 18, channels=1 << 18)
    assert conv(L, **big, tokens=1 << 20) == NO_SUPPORT
    assert conv(L, **big, sequences=1 << 13) == NO_SUPPORT


def delta(L, q=None, k=None, v=None, out=None, **kw):
    a = dict(g=P, beta=P, gs=2, a_log=None, dt=None, dk=128, dv=128, starts=None, sequences=2, tokens=6, states=R, slots=4,
             sin=P, sout=P, scale=0.1, eps=1e-6)
    a.update(kw)
    return L.exl3_hip_delta_rule(ref(q or view()), ref(k or view()), ref(v or view()), a["g"], a["beta"], a["gs"],
                                 a["a_log"], a["dt"], ref(out or view(Q)), a["dk"], a["dv"], a["starts"], a["sequences"],
                                 a["tokens"], a["states"], a["slots"], a["sin"], a["sout"], a["scale"], a["eps"], None, 0,
                                 None)


def test_delta_rule(L):
    assert delta(L, sequences=0, starts=P) == OK
    for bad in PACKED_BAD + (dict(dk=32), dict(dk=96), dict(dk=256), dict(dv=0), dict(dv=8), dict(dv=24), dict(dv=272),
                             dict(g=None), dict(beta=None), dict(g=P + 2), dict(beta=P + 1), dict(gs=1), dict(gs=1 << 41),
                             dict(gs=1 << 40, tokens=1 << 10), dict(a_log=P), dict(dt=P), dict(a_log=P + 2, dt=P),
                             dict(scale=NAN), dict(scale=INF), dict(eps=NAN), dict(eps=-INF)):
        assert delta(L, **bad) == INVAL, bad
    for x in (view(None), view(P + 1), view(heads=1), view(heads=3), view(heads=0)):
        assert delta(L, q=x) == INVAL
        assert delta(L, k=x) == INVAL
    for x in (view(None), view(P + 1), view(heads=1), view(heads=3), view(heads=0), view(heads=1025)):
        assert delta(L, v=x) == INVAL
    for out in (view(None), view(Q, heads=4), view(Q, head=64), view(P), view(Q, token=100)):
        assert delta(L, out=out) == INVAL
    big = dict(starts=P, gs=16, q=view(heads=16, token=2048), k=view(heads=16, token=2048),
               v=view(heads=16, token=2048), out=view(Q, heads=16, token=2048))
    assert delta(L, **big, tokens=1 << 21) == NO_SUPPORT  # 2^15 chunks of 2^7 slices
    assert delta(L, **big, tokens=64, sequences=1 << 15) == NO_SUPPORT
    assert delta(L, starts=P, tokens=1 << 29, q=view(heads=1), k=view(heads=1), v=view(heads=1), out=view(Q, heads=1),
                 states=None, sin=None, sout=None) == NO_SUPPORT


def test_delta_rule_workspace(L):
    f = L.exl3_hip_delta_rule_workspace_bytes
    for bad in ((0, 128, 128, 1, 64), (1025, 128, 128, 1, 64), (4, 96, 128, 1, 64), (4, 128, 24, 1, 64),
                (4, 128, 128, 65537, 64), (4, 128, 128, 1, 1 << 31), (4, 128, 128, 0, 4096), (4, 128, 128, 8, 8)):
        assert f(*bad) == 0, bad
    for few in ((4, 128, 128, 1, 15), (4, 128, 128, 9, 17)):
        assert f(*few) == 0, few
    sizes = [f(4, 128, 128, s, n) for s, n in ((1, 16), (8, 16), (8, 128), (1, 4096), (8, 4096))]
    assert sizes[0] > 0 and sizes == sorted(sizes)


def test_exports(L):
    for name in ("exl3_hip_rms_norm", "exl3_hip_short_conv", "exl3_hip_delta_rule", "exl3_hip_delta_rule_workspace_bytes"):
        assert name in conftest.load_amd().EXPORTS and getattr(L, name)
