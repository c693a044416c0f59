"""The example's attention block (EXL3 layers, norm and positions, cache, attention) against the same block in
64 bits."""
import importlib.util
import sys
from pathlib import Path

import numpy as np
import pytest

import attention_ref as ref

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "xiaomi-hexagon-exl3_amd" / "examples" / "attention_block.py"
# An EXL3 layer keeps a relative L2 of 1e-3, a rounding to fp16 2^-11.  Keys and queries of length sqrt(d) with
# errors of 1.5e-3 in any direction move a score by about 1.5e-3, so a row of attention is off by that (scores) and
# that again (values) beside its own size, twice that where errors fall together; then another layer.
TOLERANCE = 1e-2


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("attention_block", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class Plain:
    """the block in 64 bits; keys and values of decode steps come from the cache"""

    def __init__(self, block):
        import torch
        self.b = block
        h, hk, d = block.q_heads, block.kv_heads, block.head_dim

        def dense(rec, k, n):
            ids = torch.arange(n, dtype=torch.int32, device="cuda")
            return block.amd.get_rows(rec, block.bits, k, n, ids).cpu().numpy().astype(np.float64).T

        self.w = [dense(r, block.hidden, n) for r, n in
                  ((block.q_layer, h * d), (block.k_layer, hk * d), (block.v_layer, hk * d))]
        self.wo = dense(block.o_layer, h * d, block.hidden)

    def qkv(self, x, positions):
        b, x = self.b, x.cpu().numpy().astype(np.float64)
        q, k, v = ((x @ w).reshape(len(x), -1, b.head_dim) for w in self.w)
        f = b.inv_freq.cpu().numpy()
        turn = lambda t, n: ref.norm_rope(t, n.cpu().numpy(), 1e-6, positions, f, False, 1.0)[0]  # noqa: E731
        return turn(q, b.q_norm), turn(k, b.k_norm), v

    def cached(self, seq):
        import torch
        b, p = self.b, self.b.cache["page_tokens"]
        slots = torch.tensor([b.owned[seq][t // p] * p + t % p for t in range(b.length[seq])], device="cuda")
        k, v = b.amd.kv_cache_read(b.pages, slots, b.kv_heads, b.head_dim, out_dtype=torch.float32, **b.cache)
        return k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)

    def attend(self, q, k, v):  # the last query sees all keys, the one before all but one
        group = self.b.q_heads // self.b.kv_heads
        out = np.empty_like(q)
        for h in range(q.shape[1]):
            s = q[:, h] @ k[:, h // group].T / np.sqrt(self.b.head_dim)
            s[np.arange(len(k))[None] > np.arange(len(k) - len(q), len(k))[:, None]] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            out[:, h] = p / p.sum(1, keepdims=True) @ v[:, h // group]
        return out.reshape(len(q), -1) @ self.wo


def rel(got, want):
    return np.linalg.norm(got.cpu().numpy().astype(np.float64) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("cache_bits,head_dim,heads,page_tokens", [(4, 256, (4, 1), 16), (8, 128, (4, 2), 64),
                                                                   (4, 64, (8, 2), 256)])
def test_prompt_then_steps(amd, example, cache_bits, head_dim, heads, page_tokens):
    import torch
    b = example.AttentionBlock(amd, hidden=512, q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim,
                               cache_bits=cache_bits, page_tokens=page_tokens, page_count=40, rot_dim=head_dim // 2)
    plain = Plain(b)
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda n: torch.randn((n, 512), generator=g, device="cuda")  # noqa: E731
    b.prompt(draw(50), ["gone"], [50])  # its pages are used again, out of order
    lengths = [1, 77, 130]
    x = draw(sum(lengths))
    y = b.prompt(x[:78], [0, 1], lengths[:2]), b.prompt(x[78:], [2], lengths[2:])
    b.release("gone")
    at = 0
    for s, n in enumerate(lengths):
        q, k, v = plain.qkv(x[at:at + n], np.arange(n))
        got = y[s // 2][at:at + n] if s < 2 else y[1]
        assert rel(got, plain.attend(q, k, v)) < TOLERANCE, (s, n)
        at += n
    for tokens in (1, 1, 3, 1):  # three at once as a draft's check takes them
        x = draw(3 * tokens)
        order = [2, 0, 1]
        start = [b.length[s] for s in order]
        y = b.step(x, b.plan(order, tokens), tokens)
        for i, s in enumerate(order):
            rows = slice(i * tokens, (i + 1) * tokens)
            q, _, _ = plain.qkv(x[rows], start[i] + np.arange(tokens))
            assert rel(y[rows], plain.attend(q, *plain.cached(s))) < TOLERANCE, (tokens, s)


def test_pages_run_out_and_come_back(amd, example):
    import torch
    b = example.AttentionBlock(amd, hidden=256, q_heads=2, kv_heads=1, head_dim=128, page_tokens=16, page_count=3)
    x = torch.zeros((49, 256), device="cuda")
    with pytest.raises(RuntimeError, match="no free page"):
        b.prompt(x, [0], [49])
    b.release(0)
    b.prompt(x[:48], [1], [48])
    with pytest.raises(ValueError, match="has been started"):
        b.prompt(x[:1], [1], [1])


def test_example_runs(example, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["attention_block", "--sequences", "3", "--prompt", "300", "--steps", "5"])
    example.main()
    assert "outputs finite: True" in capsys.readouterr().out
