"""The example's linear-attention block (norm with residual, EXL3 layers, short convolution, delta rule, gated norm)
against the same block in 64 bits, and its captured steps."""
import importlib.util
import sys
from pathlib import Path

import numpy as np
import pytest

import linear_attention_ref as ref

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "xiaomi-hexagon-exl3_amd" / "examples" / "linear_attention_block.py"
# An EXL3 layer keeps a relative L2 of 1e-3, roundings to fp16 (layer, convolution) 2^-11 each: q, k, v and z are off by
# 1.3e-3.  The output is q times a sum of terms with k twice (written and read) and v once: 4 * 1.3e-3 where all fall
# together, the gate z another 1.3 * 1.3e-3, roundings of it and its norm 2 * 2^-11, and the output layer 1e-3.
TOLERANCE = 1e-2


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("linear_attention_block", EXAMPLE)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def f64(t):
    return t.cpu().numpy().astype(np.float64)


class Plain:
    """the block in 64 bits, with states of its own"""

    def __init__(self, b):
        import torch

        def dense(rec, k, n):
            return f64(b.amd.get_rows(rec, b.bits, k, n, torch.arange(n, dtype=torch.int32, device="cuda"))).T

        self.b = b
        self.qkv, self.z = dense(b.qkv_layer, b.hidden, b.channels), dense(b.z_layer, b.hidden, b.out_width)
        self.o = dense(b.o_layer, b.out_width, b.hidden)
        self.conv, self.delta = np.zeros(b.conv_states.shape), np.zeros(b.delta_states.shape)

    def rows(self, x, residual, lens, slots_in, slots_out):
        b, n = self.b, len(x)
        h, after, _ = ref.rms_norm(f64(x), f64(b.in_norm), b.eps, f64(residual))
        mixed, self.conv, _ = ref.short_conv(h @ self.qkv, f64(b.conv_weight), f64(b.conv_bias), True, lens, self.conv,
                                             slots_in, slots_out)
        kw = b.k_heads * b.key_dim
        q, k = (mixed[:, i * kw:(i + 1) * kw].reshape(n, b.k_heads, -1) for i in (0, 1))
        v, gates = mixed[:, 2 * kw:].reshape(n, b.v_heads, -1), h @ f64(b.gate_weight)
        o, self.delta, _, _ = ref.delta_rule(q, k, v, gates[:, :b.v_heads], gates[:, b.v_heads:], lens, b.key_dim ** -0.5,
                                             self.delta, slots_in, slots_out, f64(b.a_log), f64(b.dt_bias), b.eps)
        y, _, _ = ref.rms_norm(o, f64(b.out_norm), b.eps, gate=(h @ self.z).reshape(o.shape))
        return y.reshape(n, -1) @ self.o, after


def rel(got, want):
    return np.linalg.norm(f64(got) - want) / max(np.linalg.norm(want), 1e-30)


@pytest.mark.parametrize("k_heads,v_heads,key_dim,value_dim,width", [(2, 4, 128, 128, 4), (2, 2, 64, 64, 3),
                                                                     (1, 1, 128, 256, 2)])
def test_prompts_then_steps(amd, example, k_heads, v_heads, key_dim, value_dim, width):
    import torch
    b = example.LinearAttentionBlock(amd, hidden=512, k_heads=k_heads, v_heads=v_heads, key_dim=key_dim,
                                     value_dim=value_dim, width=width, slots=4)
    plain = Plain(b)
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda n: torch.randn((n, 512), generator=g, device="cuda")  # noqa: E731
    b.rows(draw(70), draw(70), ["gone"], [70])  # its state is used again, by a sequence that starts from zeros
    b.release("gone")
    # prompts; a second part of one beside a new one; a few rows of all
    for seqs, lens in (([0, 1], [1, 150]), ([1, 2], [64, 77]), ([2, 0, 1], [2, 3, 1])):
        x, r = draw(sum(lens)), draw(sum(lens))
        before = [b.slot.get(s, -1) for s in seqs]
        y, after = b.rows(x, r, seqs, lens)
        want, sum_ = plain.rows(x, r, lens, before, [b.slot[s] for s in seqs])
        at = 0
        for n in lens:
            assert rel(y[at:at + n], want[at:at + n]) < TOLERANCE, (seqs, lens, at)
            at += n
        assert rel(after, sum_) < 2.0 ** -23
    for tokens in (1, 1, 3):  # three at once as a draft's check takes them
        order = [2, 0, 1]
        x, r = draw(3 * tokens), draw(3 * tokens)
        y, _ = b.step(x, r, b.plan(order), tokens)
        slots = [b.slot[s] for s in order]
        want, _ = plain.rows(x, r, [tokens] * 3, slots, slots)
        for i in range(3):
            rows = slice(i * tokens, (i + 1) * tokens)
            assert rel(y[rows], want[rows]) < TOLERANCE, (tokens, i)
    for s in range(3):
        assert rel(b.delta_states[b.slot[s]], plain.delta[b.slot[s]]) < TOLERANCE
        assert rel(b.conv_states[b.slot[s]], plain.conv[b.slot[s]]) < TOLERANCE


def test_captured_steps_are_the_eager_ones(amd, example):
    """a graph's replays, with eager steps of another block between them, bit for bit"""
    import torch
    blocks = [example.LinearAttentionBlock(amd, hidden=512, k_heads=2, v_heads=4, slots=5) for _ in range(2)]
    x, zeros = torch.randn(90, 512, device="cuda"), torch.zeros(90, 512, device="cuda")
    for b in blocks:
        b.rows(x, zeros, list(range(5)), [10, 20, 30, 5, 25])
    held, plan, res = x[:5].clone(), blocks[0].plan([3, 1, 4, 0, 2]), zeros[:5].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        blocks[0].step(held, res, plan)
    torch.cuda.current_stream().wait_stream(side)
    blocks[1].step(held, res, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, after = blocks[0].step(held, res, plan)
    for i in range(4):
        held.copy_(x[5 * i:5 * i + 5])
        graph.replay()
        want, sum_ = blocks[1].step(held, res, plan)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(after, sum_), i
        for a, c in ((blocks[0].delta_states, blocks[1].delta_states), (blocks[0].conv_states, blocks[1].conv_states)):
            assert torch.equal(a, c), i


def test_states_run_out_and_come_back(amd, example):
    import torch
    b = example.LinearAttentionBlock(amd, hidden=256, k_heads=1, v_heads=1, slots=2)
    x = torch.zeros(40, 256, device="cuda")
    with pytest.raises(RuntimeError, match="no free state"):
        b.rows(x[:3], x[:3], [0, 1, 2], [1, 1, 1])
    b.rows(x[:2], x[:2], [0, 1], [1, 1])
    with pytest.raises(ValueError, match="fit the plan"):
        b.step(x[:3], x[:3], b.plan([0, 1]))
    b.release(0)
    b.rows(x[:1], x[:1], [2], [1])


def test_example_runs(example, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["linear_attention_block", "--sequences", "3", "--prompt", "300", "--steps", "5"])
    example.main()
    assert "outputs finite: True" in capsys.readouterr().out
