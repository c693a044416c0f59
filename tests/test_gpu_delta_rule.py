"""exl3_hip_delta_rule against its recurrence in 64 bits."""
import numpy as np
import pytest

import linear_attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def draw(seed, shape, sigma=1.0):
    return synth.normal(seed, int(np.prod(shape)), sigma).reshape(shape).astype(np.float32)


def cuda(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def starts_of(lens):
    import torch
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def inputs(seed, n, hk, hv, dk, dv, raw=True, norm=True):
    """q and k behind a SiLU (biased to positive products, as the block has them); without the norm of unit length"""
    q, k = (np.maximum(draw(seed + i, (n, hk, dk)), -0.2) for i in (0, 1))
    if not norm:
        q, k = (t / np.linalg.norm(t, axis=-1, keepdims=True) for t in (q, k))
    a, b = draw(seed + 2, (n, hv)), draw(seed + 3, (n, hv))
    d = dict(q=q.astype(np.float16), k=k.astype(np.float16), v=draw(seed + 4, (n, hv, dv), 0.7).astype(np.float16),
             g=a, beta=b, a_log=None, dt_bias=None)
    if raw:
        d["a_log"], d["dt_bias"] = draw(seed + 5, (hv,)), draw(seed + 6, (hv,)) - 2
    else:
        d["g"], d["beta"] = -np.exp(a - 2), (1 / (1 + np.exp(-b))).astype(np.float32)
    return d


def call(amd, d, lens, states=None, sin=None, sout=None, norm=True, packed=True, behind=0, **kw):
    """(out, states) of the call and of the recurrence, with the bounds checked"""
    import torch
    n, (hv, dv), dk = sum(lens), d["v"].shape[1:], d["q"].shape[2]
    eps = 1e-6 if norm else None
    scale = kw.pop("scale", dk ** -0.5)
    t = {}
    for name, x in d.items():
        if name in ("q", "k", "v", "g", "beta") and behind:
            x = np.concatenate([x, np.full((behind,) + x.shape[1:], np.nan, x.dtype)])
        t[name] = cuda(x)
    pool = cuda(states)
    out = torch.full((n + behind, hv, dv), 9.0, dtype=torch.float16, device="cuda")
    where = dict(starts=starts_of(lens)) if packed else dict(sequences=len(lens))
    amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], states=pool, slots_in=cuda(sin),
                   slots_out=cuda(sout), scale=scale, qk_eps=eps, out=out, **where, **kw)
    f = {k: None if x is None else x.astype(np.float64) for k, x in d.items()}
    want, after, bound, off = ref.delta_rule(
        f["q"], f["k"], f["v"], f["g"], f["beta"], lens, float(np.float32(scale)),
        None if states is None else states.astype(np.float64), sin, sout, f["a_log"], f["dt_bias"],
        None if eps is None else float(np.float32(eps)), chunk=64 if n >= max(16, (2 if packed and len(lens) > 1 else 16) * len(lens)) else None)
    assert bool((out[n:] == 9).all())
    got = out[:n].cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    top = np.nan_to_num(bound + ref.rounded(np.abs(want) + bound, "float16"))
    beyond = np.isinf(got)  # fp16 ends at 65,504: from 65,520 on a value rounds to infinity
    assert np.all((np.sign(got) * want)[beyond] + top[beyond] >= 65520)
    err = np.nan_to_num(np.abs(np.where(beyond, want, got) - want))
    print(f"  out: largest error {err.max(initial=0):.2e}, of its bound {np.max(err / np.maximum(top, 1e-30), initial=0):.2f}")
    assert np.all(err <= top)
    if states is not None:
        now = pool.cpu().numpy()
        left = np.zeros(len(states), bool)
        if sout is not None:
            left[[s for s in sout if 0 <= s < len(states)]] = True
        assert np.array_equal(now[~left], states[~left])
        assert np.array_equal(np.isnan(now), np.isnan(after))
        err = np.nan_to_num(np.abs(now - after))
        print(f"  states: largest error {err.max():.2e}, of its bound "
              f"{np.max(err / np.maximum(np.nan_to_num(off), 1e-30)[..., :]):.2f}")
        assert np.all(err <= np.nan_to_num(off) + ref.E32 * np.nan_to_num(np.abs(after)))
    return out, pool


HEADS = [(1, 1), (2, 2), (2, 6), (3, 3), (1, 5)]
DIMS = [(64, 16), (64, 64), (128, 128), (128, 48), (64, 96), (128, 256), (128, 112)]


@pytest.mark.parametrize("hk,hv", HEADS)
@pytest.mark.parametrize("dk,dv", DIMS)
def test_next_tokens(amd, hk, hv, dk, dv):
    """one to seven tokens of every sequence, each from its slot"""
    for n, seqs, raw, norm in ((1, 5, True, True), (4, 3, False, True), (7, 2, True, False)):
        d = inputs(10 * n, n * seqs, hk, hv, dk, dv, raw, norm)
        states = draw(77, (seqs + 2, hv, dk, dv), 0.5)
        slots = np.random.default_rng(n).permutation(seqs + 2)[:seqs].astype(np.int32)
        call(amd, d, [n] * seqs, states, slots, slots, norm, packed=False)


LENGTHS = [[1], [63], [64], [65], [130], [0, 1, 17, 64, 0, 200, 3], [0], [33, 0, 0, 34], [128, 128]]


@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("dk,dv,hk,hv", [(128, 128, 2, 2), (64, 96, 1, 3), (128, 48, 2, 4), (64, 64, 3, 3)])
def test_packed_prompts(amd, lens, dk, dv, hk, hv):
    for raw, norm, prior in ((True, True, True), (False, False, False)):
        d = inputs(5, sum(lens), hk, hv, dk, dv, raw, norm)
        states = draw(77, (len(lens) + 1, hv, dk, dv), 0.5)
        slots = np.random.default_rng(2).permutation(len(lens) + 1)[:len(lens)].astype(np.int32)
        call(amd, d, lens, states, slots if prior else None, slots, norm, behind=3)


@pytest.mark.parametrize("lens", [[1, 1, 1, 40, 0, 3, 90, 7, 8, 15, 16], [1] * 20 + [130], [2, 2, 2, 2], [9, 7], [64, 1],
                                  [16, 1, 1, 1, 1, 1, 1, 1, 1]], ids=str)
@pytest.mark.parametrize("dk,dv,hk,hv", [(128, 128, 1, 2), (64, 48, 2, 2)])
def test_short_and_long_sequences_together(amd, lens, dk, dv, hk, hv):
    d = inputs(21, sum(lens), hk, hv, dk, dv)
    states = draw(79, (len(lens) + 2, hv, dk, dv), 0.5)
    slots = np.random.default_rng(4).permutation(len(lens) + 2)[:len(lens)].astype(np.int32)
    call(amd, d, lens, states, slots, slots, behind=5)
    call(amd, d, lens, states, None, slots)


@pytest.mark.parametrize("dk,dv,hk,hv,seqs", [(128, 256, 4, 16, 4), (64, 256, 16, 16, 4), (128, 160, 26, 26, 4),
                                               (128, 32, 64, 64, 8), (64, 48, 32, 64, 6)])
def test_many_columns(amd, dk, dv, hk, hv, seqs):
    """1024 groups of 16 columns and more, in pairs where value_dim has them"""
    import torch
    lens = [70, 1, 9, 16, 64, 8, 0, 33][:seqs]
    d = inputs(22, sum(lens), hk, hv, dk, dv)
    states = draw(80, (seqs, hv, dk, dv), 0.5)
    slots = np.arange(seqs, dtype=np.int32)[::-1].copy()
    want, _ = call(amd, d, lens, states, slots, slots, behind=2)
    t = {k: cuda(x) for k, x in d.items()}
    wide = torch.zeros(sum(lens), hv, dv + 1, dtype=torch.float16, device="cuda")  # rows at no 16-byte places
    wide[..., 1:] = t["v"]
    out = torch.full_like(wide, 5)
    amd.delta_rule(t["q"], t["k"], wide[..., 1:], t["g"], t["beta"], t["a_log"], t["dt_bias"], starts=starts_of(lens),
                   states=cuda(states), slots_in=cuda(slots), qk_eps=1e-6, out=out[..., 1:])
    assert torch.equal(out[..., 1:], want[:sum(lens)]) and bool((out[..., 0] == 5).all())


@pytest.mark.parametrize("lens", [[1, 2, 1, 0, 1], [70, 2, 90, 0, 64]], ids=str)
def test_slots_that_are_none_or_beyond_the_pool(amd, lens):
    d = inputs(6, sum(lens), 2, 4, 128, 64)
    states = draw(78, (4, 4, 128, 64))
    call(amd, d, lens, states, np.array([4, -1, 1 << 30, 2, 1], np.int32), np.array([0, 4, -3, 3, 1], np.int32))
    call(amd, d, lens)
    call(amd, d, lens, states, np.array([1, 1, 1, 1, 1], np.int32))
    call(amd, d, lens, states, np.array([1, 1, 1, 1, -1], np.int32), np.array([0, 2, -1, 3, -1], np.int32))


@pytest.mark.parametrize("n", [5, 150])
def test_gates_at_their_ends(amd, n):
    """decays of 1 and 0 (-inf among them: the state is emptied) and nearly so, beta of 0 and 1"""
    d = inputs(8, n, 2, 2, 64, 64, raw=False)
    g = np.array([0.0, -np.inf, -1e-7, -1e30, -90.0, -150.0, -3e-3], np.float32)
    d["g"] = g[np.random.default_rng(1).integers(0, len(g), (n, 2))]
    d["beta"] = np.random.default_rng(2).integers(0, 2, (n, 2)).astype(np.float32)
    slot = np.zeros(1, np.int32)
    call(amd, d, [n], draw(3, (1, 2, 64, 64)), slot, slot)
    d["g"][:] = 0  # nothing is forgotten
    d["beta"][:] = 1
    call(amd, d, [n], draw(3, (1, 2, 64, 64)), slot, slot)


@pytest.mark.parametrize("n", [3, 140])
def test_raw_gates_at_their_ends(amd, n):
    d = inputs(9, n, 1, 2, 64, 64)
    d["g"] = np.random.default_rng(1).choice(np.array([-100, -20, 0, 20, 88, 1e4], np.float32), (n, 2))
    d["beta"] = np.random.default_rng(2).choice(np.array([-200, -20, 0, 20, 200], np.float32), (n, 2))
    d["a_log"] = np.array([-5.0, 2.5], np.float32)
    slot = np.zeros(1, np.int32)
    call(amd, d, [n], draw(3, (1, 2, 64, 64)), slot, slot)


@pytest.mark.parametrize("n", [2, 100])
@pytest.mark.parametrize("size", [1e-6, 1e4, 1e9])
def test_states_of_other_sizes(amd, n, size):
    """values and states far from 1: the products keep their bits at any of them"""
    d = inputs(11, n, 1, 1, 128, 32)
    d["v"] = (d["v"].astype(np.float32) * min(size, 1e4)).astype(np.float16)
    slot = np.zeros(1, np.int32)
    call(amd, d, [n], draw(3, (1, 1, 128, 32)) * np.float32(size), slot, slot, scale=1e-4 if size > 1 else 1.0)


@pytest.mark.parametrize("n", [3, 90])
def test_nan_stays_in_its_sequence(amd, n):
    import torch
    lens = [n, n, n]
    d = inputs(12, 3 * n, 2, 2, 64, 32)
    clean, _ = call(amd, d, lens)
    for name, what in (("q", np.nan), ("k", np.inf), ("v", np.nan), ("g", np.nan), ("beta", np.nan)):
        bad = {k: None if x is None else x.copy() for k, x in d.items()}
        bad[name][n + 1, 0] = what
        t = {k: cuda(x) for k, x in bad.items()}
        got = amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], starts=starts_of(lens),
                             qk_eps=1e-6)
        assert torch.equal(got[:n], clean[:n]) and torch.equal(got[2 * n:], clean[2 * n:]), name
        assert torch.equal(got[n:2 * n, 1], clean[n:2 * n, 1]), name  # and in its head
        assert bool(torch.isnan(got[n + 1, 0]).any()), name


def test_slices_of_wider_rows(amd):
    """q, k and v out of one row, at 16-byte places and between them; gates with a stride; out into a wider row"""
    import torch
    for n in (6, 80):
        d = inputs(13, n, 2, 4, 64, 32)
        t = {k: cuda(x) for k, x in d.items()}
        want = amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], sequences=2)
        for off in (0, 8, 1):
            row = torch.zeros(n, 2 * 128 + 128 + 16, dtype=torch.float16, device="cuda")
            q, k = row[:, off:off + 128].view(n, 2, 64), row[:, off + 128:off + 256].view(n, 2, 64)
            v = row[:, off + 256:off + 384].view(n, 4, 32)
            q.copy_(t["q"]), k.copy_(t["k"]), v.copy_(t["v"])
            gates = torch.zeros(n, 11, device="cuda")
            gates[:, 1:5], gates[:, 6:10] = t["g"], t["beta"]
            out = torch.full((n, 4, 40), 3.0, dtype=torch.float16, device="cuda")
            amd.delta_rule(q, k, v, gates[:, 1:5], gates[:, 6:10], t["a_log"], t["dt_bias"], sequences=2,
                           out=out[:, :, off:off + 32])
            assert torch.equal(out[:, :, off:off + 32], want), (n, off)
            assert bool((out[:, :, :off] == 3).all() and (out[:, :, off + 32:] == 3).all())


def test_the_same_bits_again(amd):
    import torch
    for lens in ([1] * 33, [300, 0, 65]):
        d = inputs(14, sum(lens), 2, 2, 128, 128)
        t = {k: cuda(x) for k, x in d.items()}
        runs = [amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"],
                               starts=starts_of(lens), qk_eps=1e-6) for _ in range(3)]
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_starts_that_are_no_packing(amd):
    """no row outside the views is read or written; a good sequence's rows are its own"""
    import torch
    d = inputs(15, 90, 1, 1, 64, 32)
    t = {k: cuda(x) for k, x in d.items()}
    starts = torch.tensor([-7, 3, 1, 8, 1 << 30], dtype=torch.int32, device="cuda")
    args = ("q", "k", "v", "g", "beta")
    got = amd.delta_rule(*(t[k] for k in args), t["a_log"], t["dt_bias"], starts=starts)
    alone = amd.delta_rule(*(t[k][8:] for k in args), t["a_log"], t["dt_bias"], starts=starts_of([82]))
    assert torch.equal(got[8:], alone)
