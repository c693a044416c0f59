"""64-bit restatements of the attention block (norm and positions, quantised cache, attention), written from
the formulas in include/exl3_hip.h, on numpy arrays."""
import numpy as np

GROUP = 32
H32 = np.array([[(-1.0) ** bin(i & j).count("1") for j in range(GROUP)] for i in range(GROUP)]) / np.sqrt(32.0)


def norm_rope(x, weight, eps, positions, inv_freq, interleaved, rope_scale):
    """(rows in 64 bits, |a| + |b| of each element's pair after the norm and the scale)"""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    size = np.abs(y)
    if inv_freq is not None:
        half = len(inv_freq)
        t = positions.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
        c, s = np.cos(t) * rope_scale, np.sin(t) * rope_scale
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else \
            (slice(0, half), slice(half, 2 * half))
        a, b = y[..., first].copy(), y[..., second].copy()
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * abs(rope_scale)
    return y, size


def h32_f32(x):
    """the rotation in binary32 with the butterflies' order that fixes the codes' bits"""
    y = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, GROUP).copy()
    for step in (1, 2, 4, 8, 16):
        z = y.reshape(*y.shape[:-1], GROUP // (2 * step), 2, step)
        a, b = z[..., 0, :].copy(), z[..., 1, :].copy()
        with np.errstate(invalid="ignore", over="ignore"):
            z[..., 0, :], z[..., 1, :] = a + b, a - b
    return (y * np.float32(0.17677669529663687)).reshape(x.shape)


def quantise(x, bits):
    """(codes [..., d] as stored, fp16 scales [..., d / 32]) of rows x, bit for bit"""
    half = 1 << (bits - 1)
    y = h32_f32(x).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top, low = y.max(-1), y.min(-1)
        ext = np.where(top > -low, top, low).astype(np.float32)
        raw = (ext * np.float32(-1.0 / half)).astype(np.float16)
        bits16 = (raw.view(np.uint16).astype(np.uint32) + (half - 1)) & ~np.uint32(half - 1)
        bad = ~np.isfinite(raw) | ((bits16 & 0x7fff) >= 0x7c00)
        bits16 = np.where((bits16 & 0x7fff) == 0, 0, bits16)
        scale = np.where(bad, np.uint16(0x7e00), bits16.astype(np.uint16)).view(np.float16)
        s32 = scale.astype(np.float32)
        r = np.where(s32 == 0, np.float32(0), np.float32(1) / s32).astype(np.float32)
        code = np.clip(np.rint(y * r[..., None]), -half, half - 1)
    code = np.where(np.isnan(code), 0, code)  # under a NaN scale the code does not matter
    return (code.astype(np.int32) + half).reshape(x.shape).astype(np.uint8), scale


def values(code, scale, bits):
    """rotated rows in 64 bits"""
    c = code.astype(np.float64) - (1 << (bits - 1))
    return (c.reshape(*scale.shape, GROUP) * scale.astype(np.float64)[..., None]).reshape(code.shape)


def rotate(x):
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore"):
        return (y @ H32).reshape(x.shape)


def page_parts(page, bits, heads, d, p):
    """views of one page's bytes: key codes [heads, p, d], value codes, key scales [heads, p, d / 32], value scales"""
    run, g = d * bits // 8, d // GROUP
    b = page.reshape(heads, -1)

    def codes(x):
        if bits == 8:
            return x
        return np.stack((x & 15, x >> 4), -1).reshape(*x.shape[:-1], -1)

    k = codes(b[:, :p * run].reshape(heads, p, run))
    v = b[:, p * run:2 * p * run].reshape(heads, p // 4, 16, 4, run // 16).transpose(0, 1, 3, 2, 4)
    v = codes(v.reshape(heads, p, run))
    ks = np.ascontiguousarray(b[:, 2 * p * run:2 * p * run + 2 * p * g]).view(np.float16).reshape(heads, p, g)
    vs = np.ascontiguousarray(b[:, 2 * p * run + 2 * p * g:]).view(np.float16).reshape(heads, p // 4, g, 4)
    return k, v, ks, vs.transpose(0, 1, 3, 2).reshape(heads, p, g)


def pack_page(k, v, ks, vs, bits):
    """the inverse of page_parts"""
    heads, p, d = k.shape

    def run(c):
        return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)

    kb, vb = run(k), run(v)
    n = kb.shape[-1]
    vb = vb.reshape(heads, p // 4, 4, 16, n // 16).transpose(0, 1, 3, 2, 4)
    ksb = np.ascontiguousarray(ks).view(np.uint8)
    vsb = np.ascontiguousarray(vs.reshape(heads, p // 4, 4, -1).transpose(0, 1, 3, 2)).view(np.uint8)
    return np.concatenate([a.reshape(heads, -1) for a in (kb, vb, ksb, vsb)], 1).reshape(-1)


def attend(q, k, v, ends, scale):
    """q [r, d] over k, v [n, d], row i over the first ends[i] keys, in 64 bits: (out, sum of weight * |v|,
    the largest sum |q||k| * scale among the keys a row sees, sum of exp(score - top))"""
    r, d = q.shape
    out, mass = np.zeros((r, d)), np.zeros((r, d))
    dots, total = np.zeros(r), np.ones(r)
    for i in range(r):
        n = int(max(0, min(len(k), ends[i])))
        if n == 0:
            continue
        s = (k[:n] @ q[i]) * scale
        e = np.exp(s - s.max())
        w = e / e.sum()
        out[i], mass[i] = w @ v[:n], w @ np.abs(v[:n])
        dots[i], total[i] = (np.abs(k[:n]) @ np.abs(q[i])).max() * abs(scale), e.sum()
    return out, mass, dots, total


U16 = 2.0 ** -11  # unit roundoff of fp16


def attention_bound(out, mass, dots, total, v_top, n, d):
    """Largest error of an attention row, element by element: each weight is rounded to fp16 (U16 of it, or 2^-25
    where it is subnormal, against a largest weight of at least 1) and so is the sum that divides; a score is a
    binary32 sum of d products of which the queries may be split in two fp16 parts (2^-22 of the product
    left), and its exponential is good to 2^-20; then one rounding of the result."""
    score = dots * (d * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
    rel = (2 * U16 + 2 * score)[:, None]
    return rel * mass + (n * 2.0 ** -25 * v_top / total)[:, None] + U16 * np.abs(out) + 2.0 ** -25
