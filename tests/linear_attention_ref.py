"""64-bit restatements of the linear-attention block (short convolution, gated delta rule, norms), written from the
formulas of include/exl3_hip.h, each with a bound on the error of a computation in 32 bits."""
import numpy as np

HALF_STEP = {"float16": 2.0 ** -11, "float32": 2.0 ** -24}  # largest relative error of a rounding
SMALLEST = {"float16": 2.0 ** -25, "float32": 2.0 ** -150}   # half a step of the subnormal numbers
E32 = 2.0 ** -24


def sigmoid(z):
    return np.exp(-np.logaddexp(0.0, -z))


def rounded(value, dtype):
    """bound on the rounding of `value` to the output's type"""
    return HALF_STEP[dtype] * np.abs(value) + SMALLEST[dtype]


def rms_norm(x, weight, eps, residual=None, gate=None):
    """(out, h, bound on out ahead of its rounding).  h is one rounded sum; the mean of squares is a sum of
    width terms in chains of at most width / 256 + 80 additions (a lane's runs, then lanes and waves), each off by E32;
    the root, the products and the gate's sigmoid add a few more."""
    h = x if residual is None else x + residual
    w = 1.0 if weight is None else weight
    y = h / np.sqrt(np.mean(h * h, -1, keepdims=True) + eps) * w
    steps = x.shape[-1] / 256 + 80 + 8
    if gate is not None:
        y = y * gate * sigmoid(gate)
        steps += 8 + 2
    return y, h, steps * E32 * np.abs(y) + 2.0 ** -140


def short_conv(x, weight, bias, silu, lens, states, slots_in, slots_out):
    """(y, states afterwards, bound on y ahead of its rounding) of packed rows"""
    n, c = x.shape
    w = weight.shape[1]
    y, size, after, at = np.zeros((n, c)), np.zeros((n, c)), None if states is None else states.copy(), 0
    for s, count in enumerate(lens):
        i = -1 if slots_in is None else int(slots_in[s])
        old = np.zeros((w - 1, c)) if i < 0 else states[i] if i < len(states) else np.full((w - 1, c), np.nan)
        line = np.concatenate([old, x[at:at + count]])
        for j in range(w):
            y[at:at + count] += line[j:j + count] * weight[:, j]
            size[at:at + count] += np.abs(line[j:j + count] * weight[:, j])
        o = -1 if slots_out is None else int(slots_out[s])
        if 0 <= o < (0 if states is None else len(states)):
            after[o] = line[count:]
        at += count
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    err = (w + 1) * E32 * size
    if silu:  # its slope is below 1.1
        y = y * sigmoid(y)
        err = 1.1 * err + 10 * E32 * np.abs(y)
    return y, after, err


def _norm(k, g, beta):
    """largest row sum of (1 + A)^-1, A_ij = beta_i exp(g_j+1 + .. + g_i) k_i . k_j (j < i)"""
    n = len(g)
    a = np.zeros((n, n))
    for i in range(n):
        fall = np.exp(np.cumsum(g[i:0:-1])[::-1])  # of rows 0 .. i - 1
        a[i, :i] = beta[i] * fall * (k[:i] @ k[i])
    return np.abs(np.linalg.inv(np.eye(n) + a)).sum(1).max() if np.all(np.isfinite(a)) else 1.0


def delta_rule(q, k, v, g, beta, lens, scale, states=None, slots_in=None, slots_out=None, a_log=None, dt_bias=None,
               qk_eps=None, unit=40 * E32, chunk=None):
    """(out, states afterwards, bounds on both ahead of out's rounding).  A column of S is off by e, |e| its
    2-norm.  Where 0 <= beta |k|^2 <= 2, the map e -> exp(g) (I - beta k k^T) e does not lengthen it, so a row adds
    only what it rounds itself: `unit` times the column's and the row's size.  unit: for the row-by-row
    kernel a dot product is a chain of 16 fused multiply-adds and 3 sums, then 8 roundings of factors (gates,
    lengths, u) and the fma of the update: 28 E32, and 2 |g| + 4 E32 for the decay.  In chunks (of `chunk` rows) u is
    T (beta (v - K S)): each of the four products that lead to S and out has operands of 22 bits (4 E32, and
    4 E32 for the product of their low parts, left out) and sums of at most 128 in binary32, whose errors are
    independent (16 E32): 4 * 24 E32, and T takes an error of its rows to at most ||T|| (largest row sum) times it.
    Their pairs end at 2^-40 of a power of two at most 4 times the bound on a column of U, ||T|| (max |beta v| + max (beta e^G
    |k|_1) max |S|): R's and U's (or W's) steps, over 64 keys of length 1, are 128 times that whatever is left of the
    chunk's states at its end."""
    n, h, dv = v.shape
    dk, group = q.shape[2], h // q.shape[1]
    q, k = (np.repeat(t, group, 1) for t in (q, k))
    if qk_eps is not None:
        q, k = (t / np.sqrt(np.sum(t * t, -1, keepdims=True) + qk_eps) for t in (q, k))
    if a_log is not None:
        g, beta = -np.exp(a_log) * np.logaddexp(0.0, g + dt_bias), sigmoid(beta)
    out, bound = np.zeros((n, h, dv)), np.zeros((n, h, dv))
    after = None if states is None else states.copy()
    off = None if states is None else np.zeros((len(states), h, dv))
    at = 0
    for s, count in enumerate(lens):
        i = -1 if slots_in is None else int(slots_in[s])
        S = np.zeros((h, dk, dv)) if i < 0 else states[i].copy() if i < len(states) else np.full((h, dk, dv), np.nan)
        e = np.zeros((h, dv))
        first, growth = at, np.ones((h, 1))
        for t in range(at, at + count):
            if chunk and (t - first) % chunk == 0:
                growth = np.array([[_norm(k[t:min(t + chunk, at + count), i], g[t:min(t + chunk, at + count), i],
                                          beta[t:min(t + chunk, at + count), i])] for i in range(h)])
                rows = slice(t, min(t + chunk, at + count))
                b = np.abs(beta[rows])[:, :, None]
                l1 = (b * np.exp(np.cumsum(g[rows], 0))[:, :, None] * np.abs(k[rows]).sum(-1, keepdims=True)).max(0)
                floor = 128 * 2.0 ** -38 * growth * ((b * np.abs(v[rows])).max(0) + l1 * np.abs(S).max(1))
            d = np.exp(g[t])[:, None, None]
            S = S * d
            u = beta[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
            size = np.sqrt(np.sum(S * S, 1)) + np.abs(beta[t])[:, None] * np.abs(v[t])
            S = S + k[t][:, :, None] * u[:, None, :]
            size = size + np.sqrt(np.sum(S * S, 1))
            gd = np.minimum(np.abs(np.where(np.isfinite(g[t]), g[t], 0)), 100)[:, None]
            e = d[:, :, 0] * e + (growth * unit * (2.4 if chunk else 1) + 2 * gd * E32) * size * np.maximum(1.0, np.linalg.norm(k[t], axis=-1))[:, None]
            out[t] = scale * np.einsum("hkv,hk->hv", S, q[t])
            if chunk and ((t - first) % chunk == chunk - 1 or t == at + count - 1):
                e = e + floor
            bound[t] = abs(scale) * np.linalg.norm(q[t], axis=-1)[:, None] * (e + growth * unit * (2.4 if chunk else 1) * size)
        o = -1 if slots_out is None else int(slots_out[s])
        if 0 <= o < (0 if states is None else len(states)):
            after[o], off[o] = S, e
        at += count
    return out, after, bound, None if off is None else off[:, :, None, :]
