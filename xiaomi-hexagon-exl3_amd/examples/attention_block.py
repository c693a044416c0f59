"""An attention block of EXL3 layers over a paged, quantised cache: prompts, then tokens one or a few at a time.

    python xiaomi-hexagon-exl3_amd/examples/attention_block.py [--cache-bits 4] [--sequences 8] [--prompt 2000] [--steps 32]

Every step is a call of this library: the q, k and v layers as one group, head norm and rotary positions, the cache
write, attention (of packed prompts, or of the newest tokens over the cache) and the output layer.  The weights
are random ones; the sizes are those of a layer with 8 query and 2 key heads of 256.
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


class AttentionBlock:
    """q, k, v and o layers, their head norms and one layer's cache of `page_count` pages.  Sequences are whole
    numbers that the caller picks; prompt() starts them, step() goes on with them, release() frees their pages."""

    def __init__(self, amd, hidden=2048, q_heads=8, kv_heads=2, head_dim=256, bits=4, cache_bits=4, page_tokens=256,
                 page_count=128, rot_dim=64, rope_base=1e4, max_sequences=64, max_rows=32, seed=1):
        self.amd, self.hidden, self.bits = amd, hidden, bits
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.cache = dict(bits=cache_bits, page_tokens=page_tokens)
        g = torch.Generator(device="cuda").manual_seed(seed)
        qn, kn = q_heads * head_dim, kv_heads * head_dim
        self.q_layer, self.k_layer, self.v_layer = (self._records(g, hidden, n) for n in (qn, kn, kn))
        self.o_layer = self._records(g, qn, hidden)
        self.q_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
        self.k_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
        self.inv_freq = (rope_base ** (-torch.arange(0, rot_dim, 2, device="cuda", dtype=torch.float64) / rot_dim)).float()
        self.pages = amd.new_kv_cache(page_count, kv_heads, head_dim, **self.cache)
        self.free = list(range(page_count - 1, -1, -1))
        self.owned, self.length = {}, {}
        # one workspace for all calls on one stream: the largest that any of them asks for
        need = max(amd.group_workspace_bytes(hidden, [qn, kn, kn], max_rows), amd.workspace_bytes(qn, hidden, max_rows),
                   amd.attention_cached_workspace_bytes(q_heads, kv_heads, head_dim, max_sequences, 1),
                   amd.attention_cached_workspace_bytes(q_heads, kv_heads, head_dim, max_sequences // 8, 8))
        self.workspace = amd.new_workspace(qn, hidden, max_rows, nbytes=need)

    def _records(self, g, k, n):
        packed = torch.randint(-32768, 32768, (k // 16, n // 16, 16 * self.bits), generator=g, device="cuda",
                               dtype=torch.int16)
        signs = lambda m: torch.randint(0, 2, (m,), generator=g, device="cuda") * 2.0 - 1.0  # noqa: E731
        su = signs(k).half()
        sv = (signs(n) * k ** -0.5 * (0.5 + torch.rand(n, generator=g, device="cuda"))).half()
        return self.amd.pack_records(packed, su, sv, self.bits, k, n)

    # ---- sequences and their pages
    def _extend(self, seqs, tokens):
        """pages for tokens[i] more tokens of each sequence; the slots of those tokens.  All of them or, by an exception,
        none."""
        p = self.cache["page_tokens"]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        start = [self.length.get(s, 0) for s in seqs]
        more = [max(0, -(-(at + n) // p) - len(self.owned.get(s, ()))) for s, at, n in zip(seqs, start, tokens)]
        if sum(more) > len(self.free):
            raise RuntimeError("the cache has no free page")
        slots = []
        for s, at, n, pages in zip(seqs, start, tokens, more):
            own = self.owned.setdefault(s, [])
            own += [self.free.pop() for _ in range(pages)]
            self.length[s] = at + n
            slots += [own[t // p] * p + t % p for t in range(at, at + n)]
        return slots

    def release(self, seq):
        self.free += reversed(self.owned.pop(seq, []))
        self.length.pop(seq, None)

    # ---- the steps that prompt and decode share
    def _qkv(self, x, positions):
        """queries, keys and values [tokens, heads, head_dim] in fp16, q and k normed and at their positions"""
        h, hk, d, t = self.q_heads, self.kv_heads, self.head_dim, x.shape[0]
        q, k, v = self.amd.mul_mat_group([(self.q_layer, h * d), (self.k_layer, hk * d), (self.v_layer, hk * d)],
                                         self.bits, self.hidden, x, out_dtype=torch.float16, workspace=self._ws(t))
        q, k = q.view(t, h, d), k.view(t, hk, d)
        self.amd.qk_norm_rope(q, k, positions, self.inv_freq, self.q_norm, self.k_norm, q_out=q, k_out=k)  # in place
        return q, k, v.view(t, hk, d)

    def _out(self, a):
        t, n = a.shape[0], self.q_heads * self.head_dim
        return self.amd.mul_mat(self.o_layer, self.bits, n, self.hidden, a.view(t, n), workspace=self._ws(t))

    def _ws(self, rows):  # prompts take the library's own workspace, which it grows as needed
        return self.workspace if rows <= 32 else None

    def prompt(self, x, seqs, lengths):
        """x [sum of lengths, hidden]: the tokens of new sequences, one after the other.  Attention runs over keys
        and values as computed; the cache receives them for the steps that follow.  The layers take up to 65,536
        tokens in a call.  -> [tokens, hidden]"""
        for s in seqs:
            if s in self.length:
                raise ValueError(f"sequence {s} has been started")
        slots, positions, starts = self._extend(seqs, lengths), [], [0]
        for n in lengths:
            positions += range(n)
            starts.append(starts[-1] + n)
        positions, starts = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (positions, starts))
        q, k, v = self._qkv(x, positions)
        self.amd.kv_cache_write(self.pages, k, v, torch.tensor(slots, device="cuda"), **self.cache)
        return self._out(self.amd.attention_prompt(q, k, v, starts))

    def plan(self, seqs, tokens=1):
        """the next `tokens` tokens of each sequence: (positions, slots, page table, lengths) on the GPU"""
        slots = self._extend(seqs, [tokens] * len(seqs))
        lens = [self.length[s] for s in seqs]
        wide = max(len(self.owned[s]) for s in seqs)
        table = [self.owned[s] + [-1] * (wide - len(self.owned[s])) for s in seqs]
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        return (i32([n - tokens + i for n in lens for i in range(tokens)]), torch.tensor(slots, device="cuda"),
                i32(table), i32(lens))

    def step(self, x, plan, tokens=1):
        """x [sequences * tokens, hidden], the tokens of plan() -> [sequences * tokens, hidden].  Makes no
        allocation outside torch's and no synchronisation: it can be captured in a HIP graph."""
        positions, slots, table, lens = plan
        q, k, v = self._qkv(x, positions)
        self.amd.kv_cache_write(self.pages, k, v, slots, **self.cache)
        return self._out(self.amd.attention_cached(q, self.pages, table, lens, self.kv_heads, q_len=tokens,
                                                   workspace=self.workspace, **self.cache))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--cache-bits", type=int, default=4, choices=(4, 8))
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2000, help="tokens of the longest prompt")
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    if not (1 <= a.sequences <= 32 and a.prompt >= 1 and a.steps >= 1):
        sys.exit("1..32 sequences, at least one prompt token and one step")
    lengths = [max(1, a.prompt * (i + 1) // a.sequences) for i in range(a.sequences)]
    if sum(lengths) > 65536:
        sys.exit(f"{sum(lengths)} prompt tokens: at most 65,536 go into one call")
    pages = sum((n + a.steps + 255) // 256 for n in lengths)
    block = AttentionBlock(_binding(), cache_bits=a.cache_bits, page_count=pages, max_sequences=max(8, a.sequences))
    seqs = list(range(a.sequences))
    x = torch.randn((sum(lengths), block.hidden), device="cuda")
    block.prompt(x, seqs, lengths)  # the first call loads kernels and sizes the library's workspace
    for s in seqs:
        block.release(s)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    block.prompt(x, seqs, lengths)
    torch.cuda.synchronize()
    print(f"prompt: {sum(lengths)} tokens of {a.sequences} sequences, {(time.perf_counter() - t0) * 1e6:.0f} us")

    # one graph for every step: a step's plan is copied into the captured tensors
    block.step(x[:a.sequences].clone(), plan := block.plan(seqs))
    torch.cuda.synchronize()
    wide = max(-(-(n + a.steps) // 256) for n in lengths)
    positions, slots, table, lens = plan
    table = torch.full((a.sequences, wide), -1, dtype=torch.int32, device="cuda")
    table[:, :plan[2].shape[1]] = plan[2]
    held, xs = (positions, slots, table, lens), x[:a.sequences].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.step(xs, held)
    total = 0.0
    for _ in range(a.steps - 1):
        new = block.plan(seqs)
        for to, frm in zip(held, new):
            (to[:, :frm.shape[1]] if to.dim() == 2 else to).copy_(frm)
        xs.copy_(torch.nn.functional.normalize(y, dim=1) * block.hidden ** 0.5)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        graph.replay()
        torch.cuda.synchronize()
        total += time.perf_counter() - t0
    if a.steps > 1:
        print(f"step: {a.sequences} sequences of {min(block.length.values())} to {max(block.length.values())} tokens, "
              f"{total / (a.steps - 1) * 1e6:.1f} us; outputs finite: {bool(torch.isfinite(y).all())}")


if __name__ == "__main__":
    main()
