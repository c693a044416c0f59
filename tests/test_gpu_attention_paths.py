"""Paths of the attention kernels that only some sizes take: the second kernel's join at head dimension 64, a worker's walk
beyond its first window of page-table entries, workspaces whose status word is set, and starts that do not fit the views."""
import numpy as np
import pytest

import attention_ref as ref
import synth
from test_gpu_attention import make_cache, prompt_reference, rows, run_cached

pytestmark = pytest.mark.gpu


def reference(q, kept, q_len, heads, scale):
    """the formula in 64 bits and its bound, as test_gpu_attention.cached_reference has them, a head's rows at a time"""
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    per, d = q.shape[1] // heads, q.shape[2]
    qr = ref.rotate(q.astype(np.float64))
    for s, (k, v) in enumerate(kept):
        n = len(k)
        if not n:
            continue
        seen = np.arange(n) < (n - (q_len - 1 - np.arange(q_len)))[:, None]
        some = seen.any(1)
        for h in range(q.shape[1]):
            at, kk, vv = slice(s * q_len, (s + 1) * q_len), k[:, h // per], v[:, h // per]
            score = np.where(seen, qr[at, h] @ kk.T * scale, -np.inf)
            top = np.where(some, score.max(1), 0.0)
            e = np.exp(score - top[:, None])
            total = np.where(some, e.sum(1), 1.0)
            w = e / total[:, None]
            o, mass = w @ vv, w @ np.abs(vv)
            dots = (np.abs(qr[at, h]) @ np.abs(kk).T).max(1) * abs(scale)
            b = ref.attention_bound(o, mass, dots, total, np.abs(vv).max(), n, d).reshape(q_len, -1, 32)
            o32 = np.abs(o).reshape(q_len, -1, 32)
            both = (b.sum(-1, keepdims=True) + 6 * 2.0 ** -24 * o32.sum(-1, keepdims=True)) / np.sqrt(32)
            want[at, h] = ref.rotate(o)
            bound[at, h] = np.broadcast_to(both, b.shape).reshape(q_len, d) + ref.U16 * np.abs(want[at, h]) + 2.0 ** -25
    return want, bound


# rows of a tile * units of 256 tokens * 64^2 from 2^22 on: 64 units of 16 rows
@pytest.mark.parametrize("q_len,hq,hk,bits,lens", [(9, 16, 1, 8, [17000, 0, 300, 9000, 1]), (4, 8, 2, 4, [16500, 700])])
def test_second_kernel_joins_at_64(amd, q_len, hq, hk, bits, lens):
    d, p = 64, 64
    print("  attention_cached", q_len, hq, hk, bits, lens, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(300, len(lens) * q_len, hq, d, sigma=2.0)
    want, bound = reference(q, kept, q_len, hk, d ** -0.5)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len)
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    assert np.array_equal(got, run_cached(amd, q, pages, table, lens, hk, bits, p, q_len))


@pytest.mark.parametrize("d,bits,hq,hk,q_len,lens", [(64, 4, 32, 4, 32, [33000, 500, 12000]), (128, 8, 16, 2, 64, [40000]),
                                                     (256, 4, 64, 8, 16, [700, 9, 20000])])
def test_walk_beyond_the_first_window_of_pages(amd, d, bits, hq, hk, q_len, lens):
    """64 row tiles leave four workers, each with more than the 32 tiles a wave that one window of the page table holds;
    then a page in the middle of a worker's share that is outside the cache"""
    p = 32
    print("  attention_cached", d, bits, hq, hk, q_len, lens, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(310, len(lens) * q_len, hq, d, sigma=2.0)
    want, bound = reference(q, kept, q_len, hk, d ** -0.5)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len)
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    long = int(np.argmax(lens))
    mine = slice(long * q_len, (long + 1) * q_len)
    for at in (0.23, 0.49, 0.97):
        t = table.clone()
        t[long, int(lens[long] * at) // p] = pages.shape[0] + 5
        bad = run_cached(amd, q, pages, t, lens, hk, bits, p, q_len)
        assert np.isnan(bad[mine]).all()
        others = np.ones(len(q), bool)
        others[mine] = False
        assert np.array_equal(bad[others], got[others])


@pytest.mark.parametrize("lens,hq,hk,d", [([300, 40, 7], 4, 2, 128),      # a workgroup for each unit
                                          ([3000] * 9, 8, 8, 64),         # shared out, joined by the last worker
                                          ([9000, 300], 4, 1, 256)])      # joined by a second kernel
def test_faulted_workspace_gives_nan_until_it_is_initialised(amd, lens, hq, hk, d):
    """the status word of a private workspace, set from the host"""
    bits, p = 4, 16
    pages, table, _ = make_cache(amd, lens, hk, d, bits, p)
    q = rows(320, len(lens), hq, d, sigma=2.0)
    ws = amd.new_workspace(128, 128, 1, nbytes=amd.attention_cached_workspace_bytes(hq, hk, d, len(lens)))
    call = lambda: run_cached(amd, q, pages, table, lens, hk, bits, p, 1, workspace=ws)  # noqa: E731
    want = call()
    assert np.isfinite(want).all() and not amd.workspace_faulted(ws)
    ws.view(-1)[16 << 20] = 1  # behind the exchange
    assert amd.workspace_faulted(ws)
    for _ in range(2):
        assert np.isnan(call()).all()
    amd.workspace_init(ws)
    for _ in range(2):
        assert np.array_equal(call(), want)


@pytest.mark.parametrize("qs,ks,q_span,k_span", [
    ([0, 30], [0, 4000], (0, 30), (0, 30)), ([0, 4000], [0, 30], (0, 30), (0, 30)), ([-5, 30], [-9, 30], (0, 30), (0, 30)),
    ([20, 10], [0, 30], None, None), ([0, 30], [25, 5], (0, 30), (0, 0)), ([7, 9], [28, 2 ** 31 - 1], (7, 9), (28, 30)),
    ([-2 ** 31, 3], [29, 31], (0, 3), (29, 30))], ids=str)
def test_starts_beyond_the_rows_stay_inside(amd, qs, ks, q_span, k_span):
    """starts are held to the views: the rows around them are NaN (a read shows) or keep their mark (a write shows)"""
    import torch
    n, pad, d, hq, hk = 30, 40, 64, 2, 1

    def guarded(seed, heads):
        x = rows(seed, n, heads, d)
        big = torch.full((n + 2 * pad, heads, d), float("nan"), dtype=torch.float16, device="cuda")
        big[pad:-pad] = torch.from_numpy(x).cuda()
        return x, big[pad:-pad]

    (q, qd), (k, kd), (v, vd) = guarded(330, hq), guarded(331, hk), guarded(332, hk)
    big = torch.full((n + 2 * pad, hq, d), 9.0, dtype=torch.float16, device="cuda")
    st = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (qs, ks)]
    for causal in (True, False):
        big.fill_(9.0)
        amd.attention_prompt(qd, kd, vd, st[0], st[1], causal=causal, out=big[pad:-pad])
        got = big.cpu().numpy().astype(np.float64)
        if q_span is None:
            assert np.all(got == 9.0)
            continue
        q0, q1 = q_span
        sub = q[q0:q1], k[k_span[0]:k_span[1]], v[k_span[0]:k_span[1]]
        want, bound, _ = prompt_reference(*sub, [0, q1 - q0], [0, k_span[1] - k_span[0]], causal, d ** -0.5)
        mine = got[pad + q0:pad + q1]
        assert np.all(np.abs(mine - want) <= bound)
        got[pad + q0:pad + q1] = 9.0
        assert np.all(got == 9.0)
