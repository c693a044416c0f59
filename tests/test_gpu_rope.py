"""exl3_hip_qk_norm_rope against the formula in 64 bits.  Error of an element: the angle is reduced to a turn with
an error of at most 2^-24 + 2^-25 turns (5.6e-7 rad) and v_sin / v_cos are good to 1.3e-7, so with the binary32
products and the norm's sum (256 terms: 2^-24 * (256 / 32 + 8) at most, eight in sequence then a tree) an
element is within 2e-6 of its pair's |a| + |b|; then one rounding to the output type."""
import numpy as np
import pytest

import attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def make(seed, tokens, heads, d, dtype):
    x = synth.normal(seed, tokens * heads * d, 1.5).reshape(tokens, heads, d)
    return x.astype(np.float16 if dtype == "f16" else np.float32)


def freqs(rot, base=1e4):
    return (base ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)


def check(got, want, size, dtype):
    got = got.double().cpu().numpy()
    tol = 2e-6 * size + (ref.U16 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * np.abs(want))
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) - tol))


CASES = [  # tokens, hq, hk, d, rot, pairs, norm, in, out, scale, first position
    (1, 8, 2, 256, 64, False, True, "f16", "f16", 1.0, 4095),
    (1, 1, 1, 64, 64, True, True, "f32", "f32", 1.0, 0),
    (3, 5, 1, 128, 128, False, True, "f16", "f32", 1.25, 131071),
    (17, 16, 4, 64, 48, True, False, "f32", "f16", 1.0, 100),
    (17, 16, 4, 64, 48, False, False, "f32", "f32", 1.0, 16777000),
    (5, 3, 3, 80, 32, False, True, "f16", "f16", 0.5, 77),
    (4, 2, 1, 8, 0, False, True, "f16", "f32", 1.0, 0),
    (2, 2, 2, 200, 192, True, True, "f32", "f32", 1.0, 5),
    (2, 2, 2, 24, 16, False, False, "f16", "f16", 1.0, 9),
    (1200, 20, 5, 128, 64, False, True, "f16", "f16", 1.0, 60000),
    (9000, 4, 1, 64, 64, True, True, "f32", "f16", 1.0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"t{c[0]}h{c[1]}-{c[2]}d{c[3]}r{c[4]}")
def test_matches_formula(amd, case):
    import torch
    tokens, hq, hk, d, rot, pairs, norm, xt, yt, scale, at = case
    print("  rope", case, flush=True)
    q, k = make(11, tokens, hq, d, xt), make(12, tokens, hk, d, xt)
    qw, kw = (1 + synth.normal(s, d, 0.3).astype(np.float32) for s in (13, 14))
    pos = (at + np.arange(tokens)).astype(np.int32)
    f = freqs(rot) if rot else None
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    qo, ko = amd.qk_norm_rope(dev(q), dev(k), dev(pos) if rot else None, dev(f), dev(qw) if norm else None,
                              dev(kw) if norm else None, 1e-5, pairs, scale,
                              out_dtype=torch.float16 if yt == "f16" else torch.float32)
    for x, w, y in ((q, qw, qo), (k, kw, ko)):
        want, size = ref.norm_rope(x, w if norm else None, 1e-5, pos, f, pairs, scale)
        check(y, want, size, yt)


@pytest.mark.parametrize("size", [1e-17, 1e-10, 1e15])
def test_norm_of_small_and_large_rows(amd, size):
    """without an eps, rows whose squares are near the ends of binary32"""
    import torch
    x = (synth.normal(15, 7 * 3 * 128, 1.0).reshape(7, 3, 128) * size).astype(np.float32)
    w = (1 + synth.normal(16, 128, 0.3)).astype(np.float32)
    y, _ = amd.qk_norm_rope(torch.from_numpy(x).cuda(), None, q_weight=torch.from_numpy(w).cuda(), eps=0.0,
                            out_dtype=torch.float32)
    want, mass = ref.norm_rope(x, w, 0.0, None, None, False, 1.0)
    check(y, want, mass, "f32")


@pytest.mark.parametrize("pairs", [False, True])
def test_views_in_place_and_unaligned(amd, pairs):
    """slices of a fused buffer, at an offset that is not 16-byte aligned, head-major outputs, and in place"""
    import torch
    tokens, hq, hk, d, rot = 13, 6, 2, 64, 32
    pos, f = np.arange(tokens, dtype=np.int32), freqs(rot)
    pd, fd = torch.from_numpy(pos).cuda(), torch.from_numpy(f).cuda()
    width = (hq + 2 * hk) * d + 3
    raw = synth.normal(21, tokens * width + 1, 1.0).astype(np.float16)
    buf = torch.from_numpy(raw).cuda()
    rows = buf[1:].view(tokens, width)
    q, k = rows[:, :hq * d].unflatten(1, (hq, d)), rows[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    w = torch.full((d,), 1.5, device="cuda")
    qo = torch.full((hq, tokens, d), float("nan"), dtype=torch.float16, device="cuda")
    ko = torch.full((hk, tokens, d), float("nan"), dtype=torch.float16, device="cuda")
    amd.qk_norm_rope(q, k, pd, fd, w, None, interleaved=pairs, q_out=qo.transpose(0, 1), k_out=ko.transpose(0, 1))
    host = raw[1:].reshape(tokens, width)
    for x, wt, y in ((host[:, :hq * d].reshape(tokens, hq, d), np.full(d, 1.5, np.float32), qo),
                     (host[:, hq * d:(hq + hk) * d].reshape(tokens, hk, d), None, ko)):
        want, size = ref.norm_rope(x, wt, 1e-6, pos, f, pairs, 1.0)
        check(y.transpose(0, 1), want, size, "f16")
    amd.qk_norm_rope(q, k, pd, fd, w, None, interleaved=pairs, q_out=q, k_out=k)
    assert torch.equal(q, qo.transpose(0, 1)) and torch.equal(k, ko.transpose(0, 1))
    rest = host.copy()
    assert np.array_equal(rows[:, (hq + hk) * d:].cpu().numpy(), rest[:, (hq + hk) * d:])  # nothing beyond the heads


def test_queries_alone_zero_rows_and_non_finite(amd):
    """no keys; a row of zeros (the norm's eps); NaN and Inf stay in their head"""
    import torch
    x = make(31, 3, 4, 128, "f32")
    x[0, 1] = 0
    x[1, 2, 5], x[2, 3, 7] = np.nan, np.inf
    pos, f = np.array([3, 0, 9], np.int32), freqs(128)
    w = np.ones(128, np.float32)
    q, none = amd.qk_norm_rope(torch.from_numpy(x).cuda(), None, torch.from_numpy(pos).cuda(),
                               torch.from_numpy(f).cuda(), torch.from_numpy(w).cuda())
    assert none is None
    got = q.cpu().numpy()
    assert np.all(got[0, 1] == 0)
    assert np.all(np.isnan(got[1, 2])) and np.isnan(got[2, 3]).any()
    ok = np.ones((3, 4), bool)
    ok[1, 2] = ok[2, 3] = False
    with np.errstate(invalid="ignore"):
        want, size = ref.norm_rope(x, w, 1e-6, pos, f, False, 1.0)
    assert np.isfinite(got[ok]).all()
    assert np.all(np.abs(got[ok] - want[ok]) <= 2e-6 * size[ok] + 2.0 ** -24 * np.abs(want[ok]))
    empty, _ = amd.qk_norm_rope(torch.empty((0, 4, 128), device="cuda"), None)
    assert empty.shape == (0, 4, 128)


def test_rows_beyond_32_bit_offsets(amd):
    """a view whose rows are more than 2^32 elements apart"""
    import torch
    far = (1 << 32) + 64
    buf = torch.empty(far + 64, dtype=torch.float16, device="cuda")
    x = torch.randn(2, 64, device="cuda").half()
    buf[:64], buf[far:] = x[0], x[1]
    q = buf.as_strided((2, 1, 64), (far, 64, 1))
    f = torch.from_numpy(freqs(64)).cuda()
    pos = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    want, _ = amd.qk_norm_rope(x[:, None].contiguous(), None, pos, f)
    got, _ = amd.qk_norm_rope(q, None, pos, f)
    assert torch.equal(got, want)
