"""Performance cases of the attention block around the EXL3 layers: norms and rotary positions of
queries and keys, the quantised cache, attention over that cache and attention over a prompt.

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
GROUP = 32  # elements of a head that share a scale of the cache
EPS = 1e-6


def _binding():
    name = "exl3_amd_operators"
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, ROOT / "xiaomi-hexagon-exl3_amd" / "exl3_amd.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's queries and keys: 2048 + 512 wide projections, heads of 256, a quarter of each rotated
        dict(name="rope_b1", kind="rope", tokens=1, hq=8, hk=2, d=256, rot=64, pairs=False, norm=True, x="f16",
             base=1e7, at=4000),
        # fp32 projections (ggml's dst type) of a ragged prompt, interleaved pairs, no norms
        dict(name="rope_r1237_f32", kind="rope", tokens=1237, hq=16, hk=4, d=64, rot=48, pairs=True, norm=False,
             x="f32", base=1e4, at=0),
        # a long prompt, whole heads rotated
        dict(name="rope_8192", kind="rope", tokens=8192, hq=32, hk=8, d=128, rot=128, pairs=False, norm=True, x="f16",
             base=1e6, at=0),
        # the new keys and values of eight sequences go into their pages and are read back
        dict(name="store_b8", kind="store", tokens=8, hk=2, d=256, bits=4, page=16, x="f16", spread=True),
        # a prompt of fp32 rows into an 8-bit cache
        dict(name="store_r5003_8bit", kind="store", tokens=5003, hk=4, d=64, bits=8, page=64, x="f32", spread=False),
        # a long prompt into a 4-bit cache
        dict(name="store_16384", kind="store", tokens=16384, hk=8, d=128, bits=4, page=256, x="f16", spread=False),
        # one sequence's next token, a short context: latency
        dict(name="cached_b1_1000", kind="cached", seqs=1, q_len=1, hq=8, hk=2, d=256, bits=4, page=16, longest=1000,
             ragged=False),
        # four drafted tokens of six sequences of very different lengths checked at once, 8 bits
        dict(name="cached_draft_8bit", kind="cached", seqs=6, q_len=4, hq=12, hk=4, d=64, bits=8, page=64,
             longest=6001, ragged=True),
        # sixteen long sequences, one token each
        dict(name="cached_b16_32768", kind="cached", seqs=16, q_len=1, hq=32, hk=8, d=128, bits=4, page=256,
             longest=32768, ragged=False),
        # one short prompt
        dict(name="prompt_37", kind="prompt", seqs=1, longest=37, prefix=0, hq=8, hk=2, d=256, ragged=False,
             causal=True),
        # a batch of packed prompts of different lengths, each continuing a prefix that is in hand
        dict(name="prompt_packed", kind="prompt", seqs=7, longest=2111, prefix=500, hq=16, hk=4, d=64, ragged=True,
             causal=True),
        # one long prompt
        dict(name="prompt_8192", kind="prompt", seqs=1, longest=8192, prefix=0, hq=32, hk=8, d=128, ragged=False,
             causal=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    hk = rng.choice((1, 2, 3, 4, 8))
    return hk * rng.choice((1, 2, 3, 4, 5, 8)), hk


def draw(rng):
    kind = rng.choice(("rope", "store", "cached", "cached", "prompt", "prompt"))
    hq, hk = _heads(rng)
    d = rng.choice((64, 128, 128, 256))
    bits = rng.choice((4, 4, 8))
    page = rng.choice((16, 32, 64, 256))
    x = rng.choice(("f16", "f16", "f32"))
    if kind == "rope":
        tokens = _log_int(rng, 1, min(8192, (8192 * 40 * 128) // ((hq + hk) * d)))
        rot = rng.choice((d, d, d // 2, d // 4, 48))
        return dict(kind=kind, tokens=tokens, hq=hq, hk=hk, d=d, rot=rot, pairs=rng.random() < 0.4,
                    norm=rng.random() < 0.7, x=x, base=rng.choice((1e4, 1e6, 1e7)), at=_log_int(rng, 1, 8192) - 1)
    if kind == "store":
        return dict(kind=kind, tokens=_log_int(rng, 1, min(16384, (16384 * 8 * 128) // (hk * d))), hk=hk, d=d,
                    bits=bits, page=page, x=x, spread=rng.random() < 0.5)
    if kind == "cached":
        seqs, q_len = _log_int(rng, 1, 16), rng.choice((1, 1, 1, 2, 3, 4, 7))
        most = min(32768, (16 * 32768 * 8 * 128) // (seqs * hk * d))  # no larger than the largest listed one
        return dict(kind=kind, seqs=seqs, q_len=q_len, hq=hq, hk=hk, d=d, bits=bits, page=page,
                    longest=_log_int(rng, 16, most), ragged=rng.random() < 0.5)
    seqs = rng.choice((1, 1, 2, 3, 5, 8))
    prefix = rng.choice((0, 0, _log_int(rng, 1, 1024)))
    most = math.isqrt(32 * 8192 * 8192 * 128 // (seqs * hq * max(d, 128)))
    return dict(kind=kind, seqs=seqs, longest=_log_int(rng, 1, max(1, min(8192, most) - prefix)), prefix=prefix,
                hq=hq, hk=hk, d=d, ragged=rng.random() < 0.6, causal=rng.random() < 0.8)


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


def _page_bytes(case):
    return case["hk"] * case["page"] * 2 * (case["d"] * case["bits"] // 8 + case["d"] // GROUP * 2)


def work(case):
    kind, d = case["kind"], case["d"]
    if kind == "rope":
        n = case["tokens"] * (case["hq"] + case["hk"]) * d
        return {"bytes": n * ((2 if case["x"] == "f16" else 4) + 2) + case["tokens"] * 4 + case["rot"] * 2,
                "flops": n * 8}
    if kind == "store":
        n = case["tokens"] * case["hk"] * d * 2
        packed = case["tokens"] * _page_bytes(case) // case["page"]
        return {"bytes": n * ((2 if case["x"] == "f16" else 4) + 2) + 2 * packed + case["tokens"] * 8,
                "flops": n * 14}
    lens = _lengths(case)
    if kind == "cached":
        token = _page_bytes(case) // case["page"]
        q = case["seqs"] * case["q_len"] * case["hq"] * d
        pairs = sum(max(0, n - j) for n in lens for j in range(case["q_len"]))
        return {"bytes": sum(lens) * token + 4 * q + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4 * d * case["hq"] * pairs}
    pre = case["prefix"]
    q, kv = sum(lens), sum(n + pre for n in lens)
    pairs = sum(n * pre + (n * (n + 1) // 2 if case["causal"] else n * n) for n in lens)
    return {"bytes": 4 * q * case["hq"] * d + 4 * kv * case["hk"] * d, "flops": 4 * d * case["hq"] * pairs}


# ------------------------------------------------------------------ inputs
class _Inputs:
    """Seeded inputs on the GPU, drawn in a fixed order."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed))

    def normal(self, *shape, sigma=1.0):
        return torch.randn(shape, generator=self.g, device="cuda") * sigma

    def channels(self, *shape, spread=0.5):
        """per-channel magnitudes: a few channels of a head are several times the others, as in trained keys"""
        return torch.exp(self.normal(*shape, sigma=spread))

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _starts(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _Inputs(seed)
    kind, d = case["kind"], case["d"]
    s = dict(case)
    if kind == "rope":
        hq, hk, n = case["hq"], case["hk"], case["tokens"]
        rows = (g.normal(n, hq + hk, d) * g.channels(hq + hk, d)).to(DTYPES[case["x"]])
        s["q"], s["k"] = rows[:, :hq], rows[:, hq:]  # the projections write one buffer
        s["qw"], s["kw"] = 1 + g.normal(d, sigma=0.2), 1 + g.normal(d, sigma=0.2)
        s["positions"] = (case["at"] + torch.arange(n, device="cuda")).to(torch.int32)
        i = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
        s["inv_freq"] = (case["base"] ** (-i / case["rot"])).float()
        return s
    if kind == "store":
        n, hk = case["tokens"], case["hk"]
        s["k"] = (g.normal(n, hk, d) * g.channels(hk, d)).to(DTYPES[case["x"]])
        s["v"] = g.normal(n, hk, d, sigma=0.7).to(DTYPES[case["x"]])
        pages = -(-n // case["page"]) * (4 if case["spread"] else 1) + 1
        if case["spread"]:  # tokens of many sequences: one place here, one there
            slots = g.perm(pages * case["page"])[:n]
        else:  # one prompt: whole pages in the order in which they were free
            table = g.perm(pages)
            at = torch.arange(n, device="cuda")
            slots = table[at // case["page"]] * case["page"] + at % case["page"]
        s["slots"] = slots.to(torch.int64)
        s["pages"] = torch.zeros((pages, _page_bytes(case)), dtype=torch.uint8, device="cuda")
        return s
    lens = _lengths(case)
    if kind == "cached":
        need = [max(1, -(-n // case["page"])) for n in lens]
        width, pages = max(need), sum(need)
        order = g.perm(pages).to(torch.int32)
        table = torch.zeros((case["seqs"], width), dtype=torch.int32, device="cuda")
        for i, m in enumerate(need):
            table[i, :m] = order[sum(need[:i]):sum(need[:i]) + m]
        s["table"], s["lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = g.normal(case["seqs"] * case["q_len"], case["hq"], d, sigma=2.0).half()
        s["pages"] = torch.empty((pages, _page_bytes(case)), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 25) // (case["page"] * case["hk"] * d))
        kc, mean = g.channels(case["hk"], d), g.normal(case["hk"], d, sigma=0.3)
        for at in range(0, pages, step):  # the contents of the cache, a piece of the pages at a time
            m = min(step, pages - at)
            k = g.normal(m, case["page"], case["hk"], d) * kc
            v = g.normal(m, case["page"], case["hk"], d, sigma=0.7) + mean
            s["pages"][at:at + m] = _pack(_quantise(k, case["bits"]), _quantise(v, case["bits"]), case)
        return s
    pre, n_kv = case["prefix"], [n + case["prefix"] for n in lens]
    s["q"] = g.normal(sum(lens), case["hq"], d, sigma=2.0).half()
    s["k"] = (g.normal(sum(n_kv), case["hk"], d) * g.channels(case["hk"], d)).half()
    s["v"] = (g.normal(sum(n_kv), case["hk"], d, sigma=0.7) + g.normal(case["hk"], d, sigma=0.3)).half()
    s["q_starts"], s["kv_starts"] = _starts(lens), _starts(n_kv)
    s["q_longest"], s["kv_longest"] = max(lens), case["longest"] + pre
    return s


# ------------------------------------------------------------------ plain forms
def _stage(x, step):
    """the butterflies (a, b) -> (a + b, a - b) between elements `step` apart"""
    y = x.reshape(*x.shape[:-1], GROUP // (2 * step), 2, step)
    a, b = y[..., 0, :], y[..., 1, :]
    return torch.stack((a + b, a - b), dim=-2).reshape(x.shape)


def _h32(x):
    """the orthonormal Walsh-Hadamard rotation of each 32 consecutive elements, in 32 bits"""
    y = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    y = _stage(_stage(_stage(_stage(_stage(y, 1), 2), 4), 8), 16)
    return (y * 0.17677669529663687).reshape(x.shape)


def _quantise(x, bits):
    """(stored codes uint8 [..., d], scales f16 [..., d / 32]) of rows x [..., d]: a group's scale takes its
    element of largest magnitude to the lowest code; it is rounded up to the 12 - bits significant bits with
    which every scale * code is an f16 number"""
    half = 1 << (bits - 1)
    y = _h32(x.float()).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    top, low = y.amax(-1), y.amin(-1)
    scale = (torch.where(top > -low, top, low) * (-1.0 / half)).half().view(torch.int16)
    scale = ((scale + (half - 1)) & -half).view(torch.float16)
    r = torch.where(scale == 0, torch.zeros_like(top), 1.0 / scale.float())
    code = torch.clamp(torch.round(y * r[..., None]), -half, half - 1) + half
    return code.reshape(x.shape).to(torch.uint8), scale


def _nibbles(code, bits):
    """codes [..., n] as bytes [..., n * bits / 8], the first code in the low half"""
    return code if bits == 8 else code[..., 0::2] | (code[..., 1::2] << 4)


def _pack(k, v, case):
    """page bytes [pages, page bytes] of the (codes, scales) of keys and values [pages, page, heads, ...]"""
    n, p, h, d = k[0].shape
    kc = _nibbles(k[0], case["bits"]).permute(0, 2, 1, 3).reshape(n, h, -1)
    vc = _nibbles(v[0], case["bits"]).reshape(n, p // 4, 4, h, 16, -1).permute(0, 3, 1, 4, 2, 5).reshape(n, h, -1)
    ks = k[1].permute(0, 2, 1, 3).contiguous().view(torch.uint8).reshape(n, h, -1)
    vs = v[1].reshape(n, p // 4, 4, h, d // GROUP).permute(0, 3, 1, 4, 2).contiguous().view(torch.uint8)
    return torch.cat((kc, vc, ks, vs.reshape(n, h, -1)), dim=-1).reshape(n, -1)


def _unnibble(b, bits):
    return b if bits == 8 else torch.stack((b & 15, b >> 4), dim=-1).reshape(*b.shape[:-1], -1)


def _unpack(pages, case):
    """keys and values (rotated, 32 bits) [pages, page, heads, d] of page bytes"""
    n, p, h, d, bits = pages.shape[0], case["page"], case["hk"], case["d"], case["bits"]
    half, cb, sb = 1 << (bits - 1), p * d * bits // 8, p * d // GROUP * 2
    b = pages.reshape(n, h, -1)
    kc = _unnibble(b[..., :cb].reshape(n, h, p, -1), bits)
    vc = _unnibble(b[..., cb:2 * cb].reshape(n, h, p // 4, 16, 4, -1).transpose(3, 4).reshape(n, h, p, -1), bits)
    ks = b[..., 2 * cb:2 * cb + sb].contiguous().view(torch.float16).reshape(n, h, p, d // GROUP, 1)
    vs = b[..., 2 * cb + sb:].contiguous().view(torch.float16).reshape(n, h, p // 4, d // GROUP, 4)
    vs = vs.transpose(3, 4).reshape(n, h, p, d // GROUP, 1)
    k = (kc.float() - half).reshape(n, h, p, d // GROUP, GROUP) * ks.float()
    v = (vc.float() - half).reshape(n, h, p, d // GROUP, GROUP) * vs.float()
    return k.reshape(n, h, p, d).transpose(1, 2), v.reshape(n, h, p, d).transpose(1, 2)


def _plain_rope(s):
    d, rot = s["d"], s["rot"]

    def one(x, w):
        x = x.float()
        if s["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        t = s["positions"].float()[:, None] * s["inv_freq"]
        c, sn = torch.cos(t)[:, None], torch.sin(t)[:, None]
        if s["pairs"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            turned = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).reshape(*x.shape[:-1], rot)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            turned = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
        return torch.cat((turned, x[..., rot:]), dim=-1).half()

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _plain_store(s):
    p, n = s["page"], s["tokens"]
    (kc, ks), (vc, vs) = _quantise(s["k"], s["bits"]), _quantise(s["v"], s["bits"])
    bytes_ = _pack_tokens(s, kc, ks, vc, vs)
    pages = s["pages"]
    pages.view(-1)[bytes_[0]] = bytes_[1]
    page, at = s["slots"] // p, s["slots"] % p
    # only the pages that hold the tokens, each once
    used, where = torch.unique(page, return_inverse=True)
    k, v = _unpack(pages[used], s)
    return _h32(k[where, at]).reshape(n, s["hk"], s["d"]).half(), _h32(v[where, at]).reshape(n, s["hk"], s["d"]).half()


def _pack_tokens(s, kc, ks, vc, vs):
    """(byte addresses, bytes) of the tokens' codes and scales in the pages"""
    p, hk, d, bits, n = s["page"], s["hk"], s["d"], s["bits"], s["tokens"]
    cb, sb, region = p * d * bits // 8, p * d // GROUP * 2, _page_bytes(s) // hk
    slot = s["slots"][:, None]
    base = (slot // p) * _page_bytes(s) + torch.arange(hk, device=slot.device) * region
    at = slot % p
    row = torch.arange(d * bits // 8, device=slot.device)
    part = d * bits // 128  # bytes of one of a value row's 16 slices
    pair = torch.arange(2, device=slot.device)
    grp = torch.arange(d // GROUP, device=slot.device)
    k_at = (base + at * (d * bits // 8))[..., None] + row
    v_at = (base + cb + at // 4 * (d * bits // 2) + at % 4 * part)[..., None] + row // part * (4 * part) + row % part
    ks_at = ((base + 2 * cb + at * (d // GROUP * 2))[..., None] + grp * 2)[..., None] + pair
    vs_at = ((base + 2 * cb + sb + at // 4 * (d // GROUP * 8) + at % 4 * 2)[..., None] + grp * 8)[..., None] + pair
    where = torch.cat([t.reshape(-1) for t in (k_at, v_at, ks_at, vs_at)])
    what = torch.cat([t.reshape(-1) for t in (_nibbles(kc, bits), _nibbles(vc, bits), ks.view(torch.uint8),
                                              vs.view(torch.uint8))])
    return where, what


def _softmax_rows(scores, seen):
    """softmax over the last axis among the places in `seen`; a row that sees nothing is zero"""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_cached(s):
    b, t, hq, hk, d, p = s["seqs"], s["q_len"], s["hq"], s["hk"], s["d"], s["page"]
    width = s["table"].shape[1] * p
    k, v = _unpack(s["pages"], s)
    idx = s["table"].long()
    k = k[idx].reshape(b, width, hk, d).transpose(1, 2)
    v = v[idx].reshape(b, width, hk, d).transpose(1, 2)
    q = _h32(s["q"].float()).reshape(b, t, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = (q @ k.transpose(2, 3)).reshape(b, hk, hq // hk, t, width) * d ** -0.5
    end = s["lens"][:, None] - (t - 1 - torch.arange(t, device=q.device))  # keys that token j sees
    seen = torch.arange(width, device=q.device) < end[:, None, None, :, None]
    out = _softmax_rows(scores, seen).reshape(b, hk, -1, width) @ v
    out = _h32(out).reshape(b, hk, hq // hk, t, d).permute(0, 3, 1, 2, 4)
    return out.reshape(b * t, hq, d).half()


def _padded(x, starts, longest):
    """packed rows [tokens, heads, d] as [sequences, heads, longest, d] in 32 bits, and their lengths"""
    lens = (starts[1:] - starts[:-1]).long()
    at = torch.arange(longest, device=x.device)
    idx = (starts[:-1].long()[:, None] + at).clamp(max=max(0, x.shape[0] - 1))
    return x.float()[idx].transpose(1, 2), lens


def _plain_prompt(s):
    hq, hk, d = s["hq"], s["hk"], s["d"]
    q, nq = _padded(s["q"], s["q_starts"], s["q_longest"])
    k, nk = _padded(s["k"], s["kv_starts"], s["kv_longest"])
    v, _ = _padded(s["v"], s["kv_starts"], s["kv_longest"])
    b, lq, lk = q.shape[0], q.shape[2], k.shape[2]
    scores = q.reshape(b, hk, -1, d) @ k.transpose(2, 3) * d ** -0.5
    scores = scores.reshape(b, hq, lq, lk)
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    end = nk[:, None] - nq[:, None] + i + 1 if s["causal"] else nk[:, None].expand(b, lq)
    seen = (j < end[:, :, None]) & (j < nk[:, None, None])
    out = _softmax_rows(scores, seen[:, None]).reshape(b, hk, -1, lk) @ v
    out = out.reshape(b, hq, lq, d).transpose(1, 2).half()
    return out[i[None, :] < nq[:, None]]


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["kind"]
    if not own:
        return {"rope": _plain_rope, "store": _plain_store, "cached": _plain_cached, "prompt": _plain_prompt}[kind](s)
    amd = _binding()
    if kind == "rope":
        w = (s["qw"], s["kw"]) if s["norm"] else (None, None)
        return amd.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=w[0], k_weight=w[1], eps=EPS,
                                interleaved=s["pairs"], out_dtype=torch.float16)
    if kind == "store":
        amd.kv_cache_write(s["pages"], s["k"], s["v"], s["slots"], bits=s["bits"], page_tokens=s["page"])
        return amd.kv_cache_read(s["pages"], s["slots"], s["hk"], s["d"], bits=s["bits"], page_tokens=s["page"],
                                 out_dtype=torch.float16)
    if kind == "cached":
        return amd.attention_cached(s["q"], s["pages"], s["table"], s["lens"], s["hk"], bits=s["bits"],
                                    page_tokens=s["page"], q_len=s["q_len"])
    return amd.attention_prompt(s["q"], s["k"], s["v"], s["q_starts"], s["kv_starts"], causal=s["causal"])


# ------------------------------------------------------------------ in 64 bits
def _exact_h32():
    """the rotation as a matrix: (-1)^(ones of i & j) / sqrt(32)"""
    m = np.array([[(-1.0) ** bin(i & j).count("1") for j in range(GROUP)] for i in range(GROUP)])
    return torch.from_numpy(m / math.sqrt(GROUP)).cuda()


def _rotated(x, h):
    return (x.double().unflatten(-1, (-1, GROUP)) @ h).flatten(-2)


def _exact_values(x, bits):
    """what the cache holds for rows x, back in their own basis"""
    h, half = _exact_h32(), 2 ** (bits - 1)
    y = _rotated(x, h).unflatten(-1, (-1, GROUP))
    ext = y.gather(-1, y.abs().argmax(-1, keepdim=True))
    scale = (ext / -half).half().double()
    part, power = torch.frexp(scale)  # magnitude in [1/2, 1): 12 - bits bits of it, upwards
    scale = torch.ldexp(torch.ceil(part.abs() * 2 ** (12 - bits)) / 2 ** (12 - bits) * part.sign(), power)
    code = (y / torch.where(scale == 0, 1.0, scale)).round().clamp(-half, half - 1) * (scale != 0)
    return _rotated((code * scale).flatten(-2), h)


def _exact_rows(page, case, head):
    """rotated keys and values in 64 bits of some pages' bytes [n, page bytes], one head: [n * page, d] each"""
    p, d, bits = case["page"], case["d"], case["bits"]
    n, size = page.shape[0], p * d * bits // 8
    region = page.shape[1] // case["hk"]
    mine = page[:, head * region:(head + 1) * region]

    def codes(b):
        b = b.to(torch.int16)
        if bits == 4:
            b = torch.stack((b % 16, b // 16), -1).flatten(-2)
        return b.double() - 2 ** (bits - 1)

    groups = d // GROUP
    k = codes(mine[:, :size].reshape(n, p, d * bits // 8))
    v = codes(mine[:, size:2 * size].reshape(n, p // 4, 16, 4, d * bits // 128)).permute(0, 1, 3, 2, 4).reshape(n, p, d)
    sc = mine[:, 2 * size:].contiguous().view(torch.float16).double()
    ks = sc[:, :p * groups].reshape(n, p, groups)
    vs = sc[:, p * groups:].reshape(n, p // 4, groups, 4).transpose(2, 3).reshape(n, p, groups)
    k = k * ks.repeat_interleave(GROUP, -1)
    v = v * vs.repeat_interleave(GROUP, -1)
    return k.reshape(n * p, d), v.reshape(n * p, d)


def _exact_attention(q, k, v, ends, scale):
    """rows q [r, d] over k, v [n, d]; row i sees the first ends[i] keys"""
    w = q @ k.T * scale
    w = w.masked_fill(torch.arange(k.shape[0], device=q.device)[None] >= ends[:, None], -math.inf)
    w = torch.softmax(w, -1)
    return torch.where(ends[:, None] > 0, torch.nan_to_num(w), 0.0) @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind, d = case["kind"], case["d"]
    if kind == "rope":
        f = s["inv_freq"].double()
        t = s["positions"].double()[:, None] * f
        turn = torch.polar(torch.ones_like(t), t)[:, None]
        rot, out = case["rot"], []
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            y = x.double()
            if case["norm"]:
                y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
            y = y.clone()
            first = slice(0, rot, 2) if case["pairs"] else slice(0, rot // 2)
            second = slice(1, rot, 2) if case["pairs"] else slice(rot // 2, rot)
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y)
        return tuple(out)
    if kind == "store":
        return _exact_values(s["k"], case["bits"]), _exact_values(s["v"], case["bits"])
    scale, per = 1 / math.sqrt(d), case["hq"] // case["hk"]
    if kind == "cached":
        t, h = case["q_len"], _exact_h32()
        q = _rotated(s["q"], h).reshape(case["seqs"], t, case["hk"], per, d)
        out = torch.zeros_like(q)
        for i, n in enumerate(_lengths(case)):
            used = s["pages"][s["table"][i, :-(-n // case["page"])].long()]
            ends = (n - t + 1 + torch.arange(t, device=q.device)).clamp(min=0)
            for head in range(case["hk"] if n else 0):
                k, v = _exact_rows(used, case, head)
                o = _exact_attention(q[i, :, head].reshape(t * per, d), k[:n], v[:n], ends.repeat_interleave(per), scale)
                out[i, :, head] = o.reshape(t, per, d)
        return _rotated(out, h).reshape(-1, case["hq"], d)
    out = torch.zeros((s["q"].shape[0], case["hq"], d), dtype=torch.float64, device="cuda")
    if case["hq"] * sum(n * (n + case["prefix"]) for n in _lengths(case)) > 3e9:
        return None
    qs, ks = s["q_starts"].tolist(), s["kv_starts"].tolist()
    for i in range(case["seqs"]):
        for at in range(qs[i], qs[i + 1], 2048):
            to = min(at + 2048, qs[i + 1])
            nk = ks[i + 1] - ks[i]
            ends = torch.full((to - at,), nk, device="cuda")
            if case["causal"]:
                ends = nk - (qs[i + 1] - qs[i]) + 1 + torch.arange(at - qs[i], to - qs[i], device="cuda")
            for head in range(case["hq"]):
                kv = slice(ks[i], ks[i + 1])
                out[at:to, head] = _exact_attention(s["q"][at:to, head].double(), s["k"][kv, head // per].double(),
                                                    s["v"][kv, head // per].double(), ends.clamp(min=0), scale)
    return out
