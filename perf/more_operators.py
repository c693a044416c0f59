"""Performance cases of the linear-attention block around the EXL3 layers: the short convolution with its
state, the gated delta rule of prompts and of next tokens, and the norms (with the residual's addition, or gated).

A case is a dict of plain values; `listed()` gives the fixed ones, `draw()` another of the same
ranges.  `run()` makes the binding's calls where `own` is true, and computes the same in elementary
torch operations in 32 bits where it is false.
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
CHUNK = 64  # rows that the plain form of a prompt takes at once


def _binding():
    name = "exl3_amd_more_operators"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, ROOT / "xiaomi-hexagon-exl3_amd" / "exl3_amd.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of one sequence: 16 heads of 128, state updated in place
        dict(name="delta_b1", kind="delta", seqs=1, longest=1, ragged=False, hk=16, hv=16, dk=128, dv=128, raw=True,
             norm=True, prior=True),
        # six sequences check four drafted tokens each, two value heads to a key head, gates worked out beforehand
        dict(name="delta_draft", kind="delta", seqs=6, longest=4, ragged=False, hk=4, hv=8, dk=64, dv=96, raw=False,
             norm=False, prior=True),
        # one decode step of sixty-four sequences: the states' bytes count
        dict(name="delta_b64", kind="delta", seqs=64, longest=1, ragged=False, hk=16, hv=16, dk=128, dv=128, raw=True,
             norm=True, prior=True),
        # a batch of packed prompts of different lengths that go on from kept states
        dict(name="delta_packed", kind="delta", seqs=7, longest=2111, ragged=True, hk=4, hv=8, dk=128, dv=128,
             raw=True, norm=True, prior=True),
        # one long prompt
        dict(name="delta_8192", kind="delta", seqs=1, longest=8192, ragged=False, hk=16, hv=16, dk=128, dv=128,
             raw=True, norm=True, prior=False),
        # the next token of eight sequences through the convolution of q, k and v
        dict(name="conv_b8", kind="conv", seqs=8, longest=1, ragged=False, channels=6144, width=4, x="f16", silu=True,
             bias=False, prior=True),
        # packed fp32 prompts, an odd channel count, three taps and a bias
        dict(name="conv_packed_f32", kind="conv", seqs=5, longest=1237, ragged=True, channels=1531, width=3, x="f32",
             silu=False, bias=True, prior=True),
        # a long prompt
        dict(name="conv_8192", kind="conv", seqs=1, longest=8192, ragged=False, channels=6144, width=4, x="f16",
             silu=True, bias=False, prior=False),
        # one token's norm ahead of a layer, with the residual's addition
        dict(name="norm_b1", kind="norm", tokens=1, heads=1, width=2048, x="f32", residual="f32", gate=False, y="f16"),
        # the gated norm of each head behind the delta rule
        dict(name="norm_gated_r1237", kind="norm", tokens=1237, heads=16, width=128, x="f16", residual="none",
             gate=True, y="f16"),
        # rows of an odd width
        dict(name="norm_r777_odd", kind="norm", tokens=777, heads=1, width=1531, x="f32", residual="f16", gate=False,
             y="f32"),
        # a long prompt's norm with the residual's addition
        dict(name="norm_16384", kind="norm", tokens=16384, heads=1, width=2048, x="f16", residual="f32", gate=False,
             y="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("delta", "delta", "delta", "conv", "norm"))
    if kind == "delta":
        hk = rng.choice((1, 2, 4, 8, 16))
        hv = hk * rng.choice((1, 1, 2, 3, 4))
        dk, dv = rng.choice((64, 128, 128)), rng.choice((64, 96, 128, 128, 256))
        same = dict(kind=kind, hk=hk, hv=hv, dk=dk, dv=dv, raw=rng.random() < 0.7, norm=rng.random() < 0.8,
                    prior=rng.random() < 0.7)
        one = hv * dk * dv  # a token's work; no more of it than in the largest listed ones
        if rng.random() < 0.5:
            n = rng.choice((1, 1, 1, 2, 3, 5, 8))
            return dict(seqs=_log_int(rng, 1, max(1, min(64, (64 << 18) // one))), longest=n, ragged=False, **same)
        seqs = rng.choice((1, 1, 2, 3, 5, 9))
        most = min(8192, (8192 << 18) // (one * seqs))
        return dict(seqs=seqs, longest=_log_int(rng, 1, max(1, most)), ragged=rng.random() < 0.6, **same)
    x = rng.choice(("f16", "f16", "f32"))
    if kind == "conv":
        channels = rng.choice((_log_int(rng, 1, 8192), 128 * _log_int(rng, 1, 64)))
        seqs = rng.choice((1, 1, 2, 5, 16, 64))
        most = min(8192, (8192 * 6144) // (channels * seqs * (2 if x == "f32" else 1)))
        return dict(kind=kind, seqs=seqs, longest=_log_int(rng, 1, max(1, most)), ragged=rng.random() < 0.6,
                    channels=channels, width=rng.choice((2, 3, 4, 4)), x=x, silu=rng.random() < 0.7,
                    bias=rng.random() < 0.4, prior=rng.random() < 0.7)
    gate = rng.random() < 0.4
    heads = rng.choice((1, 2, 8, 16)) if gate else 1
    width = rng.choice((64, 128, 256)) if gate else rng.choice((_log_int(rng, 1, 16384), 128 * _log_int(rng, 1, 128)))
    most = min(16384, (16384 * 2048) // (width * heads * 2))
    return dict(kind=kind, tokens=_log_int(rng, 1, max(1, most)), heads=heads, width=width, x=x,
                residual="none" if gate else rng.choice(("none", "f16", "f32")), gate=gate,
                y=rng.choice(("f16", "f16", "f32")))


def _lengths(case):
    """Tokens of each sequence: the longest first; ragged ones fall off to a hundredth, and the last of four or
    more is an empty place of the batch."""
    n, longest = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    out = [max(1, round(longest * 0.01 ** (((i * 0.6180339887) % 1.0)))) for i in range(n)]
    if n >= 4:
        out[-1] = 0
    return out


def _size(t):
    return {"f16": 2, "f32": 4, "none": 0}[t]


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["tokens"] * case["heads"] * case["width"]
        each = _size(case["x"]) * (2 if case["gate"] else 1) + 2 * _size(case["residual"]) + _size(case["y"])
        return {"bytes": n * each + 4 * case["width"], "flops": n * (9 if case["gate"] else 5)}
    lens, kept = _lengths(case), (2 if case["prior"] else 1)  # states are read where there are any, and written
    tokens = sum(lens)
    if kind == "conv":
        c, w, size = case["channels"], case["width"], _size(case["x"])
        return {"bytes": tokens * c * 2 * size + case["seqs"] * (w - 1) * c * size * kept + c * w * 4,
                "flops": tokens * c * (2 * w + 4)}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    return {"bytes": tokens * (2 * 2 * (hk * dk + hv * dv) + 8 * hv) + case["seqs"] * hv * dk * dv * 4 * kept,
            "flops": tokens * hv * dk * dv * 7}


# ------------------------------------------------------------------ inputs
class _Inputs:
    """Seeded inputs on the GPU, drawn in a fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, sigma=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * sigma

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def channels(self, *shape, spread=0.5):
        """per-channel magnitudes: a few channels are several times the others, as in trained layers"""
        return torch.exp(self.normal(*shape, sigma=spread))

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _packing(s, g, case):
    """starts (None where every sequence has as many rows) and the slots of the sequences, spread over a pool"""
    lens = _lengths(case)
    s["lens"], s["tokens"] = lens, sum(lens)
    s["starts"] = None
    if case["ragged"]:
        s["starts"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
    s["slots"] = g.perm(case["seqs"]).to(torch.int32)


def prepare(case, seed):
    g = _Inputs(seed)
    s = dict(case)
    if case["kind"] == "norm":
        t, h, w = case["tokens"], case["heads"], case["width"]
        s["x_"] = (g.normal(t, h, w) * g.channels(h, w)).to(DTYPES[case["x"]])
        s["weight"] = 1 + g.normal(w, sigma=0.2)
        s["res"] = (g.normal(t, h, w, sigma=3.0) * g.channels(h, w)).to(DTYPES[case["residual"]]) \
            if case["residual"] != "none" else None
        s["gate_"] = g.normal(t, h, w).to(DTYPES[case["x"]]) if case["gate"] else None
        return s
    _packing(s, g, case)
    n, seqs = s["tokens"], case["seqs"]
    if case["kind"] == "conv":
        c, w = case["channels"], case["width"]
        s["x_"] = (g.normal(n, c) * g.channels(c)).to(DTYPES[case["x"]])
        s["weight"] = g.normal(c, w, sigma=w ** -0.5)
        s["bias_"] = g.normal(c, sigma=0.2) if case["bias"] else None
        s["states"] = g.normal(seqs, w - 1, c).to(DTYPES[case["x"]])
        return s
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    # behind the convolution's SiLU, one row holds q, k and v
    rows = torch.nn.functional.silu(g.normal(n, 2 * hk * dk + hv * dv) * g.channels(2 * hk * dk + hv * dv, spread=0.3))
    if not case["norm"]:  # rows of about unit length, as a layer that norms by itself leaves them
        rows[:, :2 * hk * dk] *= dk ** -0.5
    rows = rows.half()
    s["q"] = rows[:, :hk * dk].view(n, hk, dk)
    s["k"] = rows[:, hk * dk:2 * hk * dk].view(n, hk, dk)
    s["v"] = rows[:, 2 * hk * dk:].view(n, hv, dv)
    a_log = torch.log(0.05 + 15.95 * g.uniform(hv))
    dt = torch.exp(math.log(1e-3) + math.log(100.0) * g.uniform(hv))
    dt_bias = dt + torch.log(-torch.expm1(-dt))  # softplus of it is dt
    a, b = g.normal(n, hv), g.normal(n, hv)
    if case["raw"]:
        s["g"], s["beta"], s["a_log"], s["dt_bias"] = a, b, a_log, dt_bias
    else:
        s["g"] = -torch.exp(a_log) * torch.nn.functional.softplus(a + dt_bias)
        s["beta"], s["a_log"], s["dt_bias"] = torch.sigmoid(b), None, None
    s["states"] = g.normal(seqs, hv, dk, dv, sigma=0.3)
    return s


# ------------------------------------------------------------------ plain forms
def _places(s):
    """(row of each place of [sequences, longest], whether it is one): packed rows as a padded batch"""
    lens = torch.tensor(s["lens"], device="cuda")
    first = torch.cumsum(lens, 0) - lens
    at = torch.arange(s["longest"], device="cuda")
    return (first[:, None] + at).clamp(max=s["tokens"] - 1), at < lens[:, None]


def _gates(s):
    g, beta = s["g"], s["beta"]
    if s["a_log"] is not None:
        g = g + s["dt_bias"]
        g = -torch.exp(s["a_log"]) * (torch.clamp(g, min=0) + torch.log1p(torch.exp(-torch.abs(g))))
        beta = 1 / (1 + torch.exp(-beta))
    return g, beta


def _unit(x, s):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS) if s["norm"] else x


def _steps(q, k, v, g, beta, state):
    """the recurrence, row by row: [sequences, heads, rows, d]"""
    out = torch.empty_like(v)
    for t in range(q.shape[2]):
        state = state * torch.exp(g[:, :, t])[..., None, None]
        kt = k[:, :, t, :, None]
        u = (v[:, :, t] - (state * kt).sum(-2)) * beta[:, :, t, None]
        state = state + kt * u[:, :, None, :]
        out[:, :, t] = (state * q[:, :, t, :, None]).sum(-2)
    return out, state


def _chunks(q, k, v, g, beta, state):
    """the same in chunks of rows: everything that does not need the state for all chunks at once"""
    b, h, n, dk = k.shape
    pad = -n % CHUNK
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, pad)) for x in (q, k, v))
    g, beta = (torch.nn.functional.pad(x, (0, pad)) for x in (g, beta))
    m = (n + pad) // CHUNK
    q, k, v = (x.reshape(b, h, m, CHUNK, -1) for x in (q, k, v))
    g, beta = (x.reshape(b, h, m, CHUNK) for x in (g, beta))
    total = torch.cumsum(g.double(), -1)
    at = torch.arange(CHUNK, device=q.device)
    lower = at[:, None] >= at
    fall = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf)).float()
    a = (k @ k.transpose(-1, -2)) * fall * beta[..., None] * (at[:, None] > at)
    t = torch.eye(CHUNK, device=q.device).expand_as(a).clone()  # (1 + a)^-1, row after row
    for i in range(1, CHUNK):
        t[..., i, :i] = -(a[..., i:i + 1, :i] @ t[..., :i, :i]).squeeze(-2)
    p = (q @ k.transpose(-1, -2)) * fall
    since, until = torch.exp(total).float()[..., None], torch.exp(total[..., -1:] - total).float()[..., None]
    kd, qd, ku = k * since, q * since, k * until
    out = torch.empty_like(v)
    for c in range(m):
        u = t[:, :, c] @ ((v[:, :, c] - kd[:, :, c] @ state) * beta[:, :, c, :, None])
        out[:, :, c] = qd[:, :, c] @ state + p[:, :, c] @ u
        state = state * since[:, :, c, -1:] + ku[:, :, c].transpose(-1, -2) @ u
    return out.reshape(b, h, n + pad, -1)[:, :, :n], state


def _plain_delta(s):
    hk, hv, dk = s["hk"], s["hv"], s["dk"]
    rows, real = _places(s)
    g, beta = _gates(s)
    q = (_unit(s["q"].float(), s) * dk ** -0.5).repeat_interleave(hv // hk, 1)
    k = _unit(s["k"].float(), s).repeat_interleave(hv // hk, 1)
    q, k, v = (x[rows].transpose(1, 2) for x in (q, k, s["v"].float()))
    g, beta = (x[rows].masked_fill(~real[..., None], 0).transpose(1, 2) for x in (g, beta))
    slots = s["slots"].long()
    state = s["states"][slots] if s["prior"] else torch.zeros_like(s["states"])
    out, state = (_steps if s["longest"] <= 16 else _chunks)(q, k, v, g, beta, state)
    s["states"][slots] = state
    return {"out": out.transpose(1, 2)[real].half(), "states": s["states"]}


def _plain_conv(s):
    w, n = s["width"], s["longest"]
    rows, real = _places(s)
    slots = s["slots"].long()
    old = s["states"][slots] if s["prior"] else torch.zeros_like(s["states"])
    x = torch.cat((old, s["x_"][rows]), dim=1).float()  # [sequences, w - 1 + rows, channels]
    y = sum(x[:, j:j + n] * s["weight"][:, j] for j in range(w))
    if s["bias"]:
        y = y + s["bias_"]
    if s["silu"]:
        y = y / (1 + torch.exp(-y))
    last = real.sum(1)[:, None] + torch.arange(w - 1, device=x.device)
    s["states"][slots] = x.gather(1, last[..., None].expand(-1, -1, x.shape[2])).to(s["states"].dtype)
    return {"out": y[real].to(s["x_"].dtype), "states": s["states"]}


def _plain_norm(s):
    h = s["x_"].float()
    if s["res"] is not None:
        h = h + s["res"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"]
    if s["gate"]:
        z = s["gate_"].float()
        y = y * (z / (1 + torch.exp(-z)))
    y = y.to(DTYPES[s["y"]])
    return y if s["res"] is None else (y, h.to(s["res"].dtype))


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["kind"]
    if not own:
        return {"delta": _plain_delta, "conv": _plain_conv, "norm": _plain_norm}[kind](s)
    amd = _binding()
    if kind == "norm":
        return amd.rms_norm(s["x_"], s["weight"], residual=s["res"], gate=s["gate_"], eps=EPS,
                            out_dtype=DTYPES[s["y"]])
    places = dict(starts=s["starts"], sequences=s["seqs"], states=s["states"],
                  slots_in=s["slots"] if s["prior"] else None, slots_out=s["slots"])
    if kind == "conv":
        out = amd.short_conv(s["x_"], s["weight"], bias=s["bias_"], silu=s["silu"], **places)
    else:
        out = amd.delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], a_log=s["a_log"], dt_bias=s["dt_bias"],
                             qk_eps=EPS if s["norm"] else None, **places)
    return {"out": out, "states": s["states"]}


# ------------------------------------------------------------------ in 64 bits
def _exact_delta(s):
    """the definition, a token of every sequence at a time"""
    hv, group = s["hv"], s["hv"] // s["hk"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    if s["norm"]:
        q, k = (x / torch.sqrt(x.square().sum(-1, keepdim=True) + EPS) for x in (q, k))
    head = torch.arange(hv, device="cuda") // group
    g, beta = s["g"].double(), s["beta"].double()
    if s["raw"]:
        g = -s["a_log"].double().exp() * torch.logaddexp(g + s["dt_bias"].double(), torch.zeros_like(g))
        beta = torch.sigmoid(beta)
    decay = g.exp()
    states, out = s["states"].double(), torch.empty_like(v)
    lens = s["lens"]
    first = np.cumsum([0] + lens)
    order = sorted(range(s["seqs"]), key=lambda i: -lens[i])  # the sequences that still have a token come first
    mem = states[s["slots"].long()[order]] if s["prior"] else torch.zeros_like(states)
    for t in range(s["longest"]):
        live = sum(n > t for n in lens)
        at = torch.tensor([int(first[i]) + t for i in order[:live]], device="cuda")
        kt = k[at][:, head]
        m = mem[:live].mul_(decay[at][..., None, None])
        err = v[at] - torch.matmul(kt[:, :, None, :], m)[:, :, 0]
        m += kt[..., None] * (beta[at][..., None] * err)[:, :, None, :]
        out[at] = torch.matmul(q[at][:, head][:, :, None, :], m)[:, :, 0] / math.sqrt(s["dk"])
    states[s["slots"].long()[order]] = mem
    return {"out": out, "states": states}


def _exact_conv(s):
    """one sequence at a time, the taps from the newest row backwards"""
    x, w, states = s["x_"].double(), s["weight"].double(), s["states"].double()
    out, at, taps = torch.zeros_like(x), 0, s["width"]
    for n, slot in zip(s["lens"], s["slots"].tolist()):
        old = states[slot].clone() if s["prior"] else torch.zeros_like(states[slot])
        line = torch.vstack((old, x[at:at + n]))
        for back in range(taps):
            out[at:at + n] += line[taps - 1 - back:taps - 1 - back + n] * w[:, taps - 1 - back]
        states[slot] = line[line.shape[0] - (taps - 1):]
        at += n
    if s["bias"]:
        out += s["bias_"].double()
    return {"out": out * torch.sigmoid(out) if s["silu"] else out, "states": states}


def _exact_norm(s):
    h = s["x_"].double() if s["res"] is None else s["x_"].double() + s["res"].double()
    y = s["weight"].double() * h / torch.sqrt(h.square().sum(-1, keepdim=True) / s["width"] + EPS)
    if s["gate"]:
        z = s["gate_"].double()
        y = y * z * torch.sigmoid(z)
    return y if s["res"] is None else (y, h)


def exact(case, seed):
    s = prepare(case, seed)
    return {"delta": _exact_delta, "conv": _exact_conv, "norm": _exact_norm}[case["kind"]](s)
