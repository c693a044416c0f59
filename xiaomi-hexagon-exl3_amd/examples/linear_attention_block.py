"""A linear-attention block of EXL3 layers with its sequences' states: packed rows of prompts, then tokens one or a few
at a time.

    python xiaomi-hexagon-exl3_amd/examples/linear_attention_block.py [--sequences 8] [--prompt 2000] [--steps 32]

Every step is a call of this library but the two small projections of the gates: the norm of the hidden state with
the residual's addition, the layers of q, k, v and of the output's gate as one group, the short convolution over q, k
and v, the gated delta rule, its gated norm and the output layer.  The weights are random ones; the sizes are
those of a layer with 16 heads of 128.
"""
import argparse
import importlib.util
import sys
import time
from pathlib import Path

import torch


def _binding():
    spec = importlib.util.spec_from_file_location("exl3_amd", Path(__file__).resolve().parents[1] / "exl3_amd.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class LinearAttentionBlock:
    """The layers, and the states of up to `slots` sequences.  Sequences are names that the caller picks: rows() starts
    those that are new and goes on with the others, step() goes on with all of a plan(), release() frees their states."""

    def __init__(self, amd, hidden=2048, k_heads=16, v_heads=16, key_dim=128, value_dim=128, width=4, bits=4, slots=64,
                 eps=1e-6, max_rows=32, seed=1):
        self.amd, self.hidden, self.bits, self.eps = amd, hidden, bits, eps
        self.k_heads, self.v_heads, self.key_dim, self.value_dim = k_heads, v_heads, key_dim, value_dim
        g = torch.Generator(device="cuda").manual_seed(seed)
        draw = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.channels, self.out_width = 2 * k_heads * key_dim + v_heads * value_dim, v_heads * value_dim
        self.qkv_layer, self.z_layer = (self._records(g, hidden, n) for n in (self.channels, self.out_width))
        self.o_layer = self._records(g, self.out_width, hidden)
        self.gate_weight = draw(hidden, 2 * v_heads) * hidden ** -0.5  # of g and beta, fp32 as they are few
        self.a_log, self.dt_bias = draw(v_heads), draw(v_heads) - 2
        self.conv_weight, self.conv_bias = draw(self.channels, width) * width ** -0.5, 0.1 * draw(self.channels)
        self.in_norm, self.out_norm = 1 + 0.1 * draw(hidden), 1 + 0.1 * draw(value_dim)
        self.conv_states = amd.new_conv_states(slots, self.channels, width)
        self.delta_states = amd.new_delta_states(slots, v_heads, key_dim, value_dim)
        self.free, self.slot = list(range(slots - 1, -1, -1)), {}
        need = max(amd.group_workspace_bytes(hidden, [self.channels, self.out_width], max_rows),
                   amd.workspace_bytes(self.out_width, hidden, max_rows))
        self.max_rows = max_rows
        self.workspace = amd.new_workspace(self.out_width, hidden, max_rows, nbytes=need)

    def _records(self, g, k, n):
        packed = torch.randint(-32768, 32768, (k // 16, n // 16, 16 * self.bits), generator=g, device="cuda",
                               dtype=torch.int16)
        signs = lambda m: torch.randint(0, 2, (m,), generator=g, device="cuda") * 2.0 - 1.0  # noqa: E731
        su = signs(k).half()
        sv = (signs(n) * k ** -0.5 * (0.5 + torch.rand(n, generator=g, device="cuda"))).half()
        return self.amd.pack_records(packed, su, sv, self.bits, k, n)

    # ---- sequences and their states
    def _take(self, seqs):
        """(slots that the sequences start from, slots that they leave their states in); all of them or, by an
        exception, none"""
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        if sum(s not in self.slot for s in seqs) > len(self.free):
            raise RuntimeError("no free state")
        from_ = [self.slot.get(s, -1) for s in seqs]  # -1: zeros
        for s in seqs:
            if s not in self.slot:
                self.slot[s] = self.free.pop()
        return from_, [self.slot[s] for s in seqs]

    def release(self, seq):
        if seq in self.slot:
            self.free.append(self.slot.pop(seq))

    # ---- the block
    def _block(self, x, residual, where, ws):
        amd, t = self.amd, x.shape[0]
        h, residual = amd.rms_norm(x, self.in_norm, residual=residual, eps=self.eps, out_dtype=torch.float16)
        mixed, z = amd.mul_mat_group([(self.qkv_layer, self.channels), (self.z_layer, self.out_width)], self.bits,
                                     self.hidden, h, out_dtype=torch.float16, workspace=ws)
        gates = torch.mm(h.float(), self.gate_weight)
        mixed = amd.short_conv(mixed, self.conv_weight, self.conv_bias, states=self.conv_states, **where)
        kw, vh, vd = self.k_heads * self.key_dim, self.v_heads, self.value_dim
        q, k = (mixed[:, i * kw:(i + 1) * kw].unflatten(1, (self.k_heads, self.key_dim)) for i in (0, 1))
        o = amd.delta_rule(q, k, mixed[:, 2 * kw:].unflatten(1, (vh, vd)), gates[:, :vh], gates[:, vh:], self.a_log,
                           self.dt_bias, states=self.delta_states, qk_eps=self.eps, **where)
        o = amd.rms_norm(o, self.out_norm, gate=z.view(t, vh, vd), eps=self.eps)
        return amd.mul_mat(self.o_layer, self.bits, self.out_width, self.hidden, o.view(t, -1), workspace=ws), residual

    def rows(self, x, residual, seqs, lengths):
        """x, residual fp32 [sum of lengths, hidden]: lengths[i] rows of each sequence, one after the other -> (the
        block's output, x + residual), both [rows, hidden].  The layers take up to 65,536 rows in a call.  Where it fails,
        new sequences stay new: their slots hold states of others."""
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        from_, to = self._take(seqs)
        try:
            if len(lengths) != len(seqs) or min(lengths, default=0) < 0 or starts[-1] != x.shape[0]:
                raise ValueError("lengths: one a sequence, together the rows of x")
            i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
            where = dict(starts=i32(starts), sequences=len(seqs), slots_in=i32(from_), slots_out=i32(to))
            return self._block(x, residual, where, self.workspace if starts[-1] <= self.max_rows else None)
        except BaseException:
            for s, was in reversed(list(zip(seqs, from_))):
                if was < 0:
                    self.release(s)
            raise

    def plan(self, seqs):
        """for step(): the slots of sequences that rows() has started, on the GPU"""
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        return torch.tensor([self.slot[s] for s in seqs], dtype=torch.int32, device="cuda")

    def step(self, x, residual, plan, tokens=1):
        """x, residual [sequences * tokens, hidden], up to max_rows rows and 15 tokens a sequence, as rows() returns it.
        Makes no allocation outside torch's and no synchronisation: it can be captured in a HIP graph."""
        where = dict(sequences=plan.shape[0], slots_in=plan, slots_out=plan)
        if x.shape[0] != plan.shape[0] * tokens or x.shape[0] > self.max_rows or not 1 <= tokens <= 15:
            raise ValueError("rows do not fit the plan")
        return self._block(x, residual, where, self.workspace)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2000, help="tokens of the longest prompt")
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    if not (1 <= a.sequences <= 32 and a.prompt >= 1 and a.steps >= 1):
        sys.exit("1..32 sequences, at least one prompt token and one step")
    lengths = [max(1, a.prompt * (i + 1) // a.sequences) for i in range(a.sequences)]
    if sum(lengths) > 65536:
        sys.exit(f"{sum(lengths)} prompt tokens: at most 65,536 go into one call")
    block = LinearAttentionBlock(_binding(), slots=a.sequences)
    seqs = list(range(a.sequences))
    x = torch.randn((sum(lengths), block.hidden), device="cuda")
    zeros = torch.zeros_like(x)
    block.rows(x, zeros, seqs, lengths)  # the first call loads kernels and sizes the library's workspace
    for s in seqs:
        block.release(s)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    block.rows(x, zeros, seqs, lengths)
    torch.cuda.synchronize()
    print(f"prompt: {sum(lengths)} tokens of {a.sequences} sequences, {(time.perf_counter() - t0) * 1e6:.0f} us")

    plan = block.plan(seqs)
    xs, residual = x[:a.sequences].clone(), zeros[:a.sequences].clone()
    block.step(xs, residual, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, after = block.step(xs, residual, plan)
    total = 0.0
    for i in range(a.steps):
        if i:
            xs.copy_(y)
            residual.copy_(after)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        graph.replay()
        torch.cuda.synchronize()
        total += time.perf_counter() - t0
    print(f"step: {a.sequences} sequences, {total / a.steps * 1e6:.1f} us; outputs finite: "
          f"{bool(torch.isfinite(y).all() and torch.isfinite(block.delta_states).all())}")


if __name__ == "__main__":
    main()
