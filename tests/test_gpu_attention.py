"""Attention over the cache and over packed prompts against the formula in 64 bits, element by element within
attention_ref.attention_bound (derived from the roundings that the entry points state)."""
import numpy as np
import pytest

import attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def rows(seed, *shape, sigma=1.0):
    return synth.normal(seed, int(np.prod(shape)), sigma).reshape(shape).astype(np.float16)


# ------------------------------------------------------------------ prompts
def prompt_reference(q, k, v, qs, ks, causal, scale):
    """(want, bound, which rows belong to a sequence)"""
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    used = np.zeros(q.shape[0], bool)
    per = q.shape[1] // k.shape[1]
    d = q.shape[2]
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    for s in range(len(qs) - 1):
        nq, nk = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        i = np.arange(nq)
        ends = nk - (nq - 1 - i) if causal else np.full(nq, nk)
        used[qs[s]:qs[s + 1]] = True
        for h in range(q.shape[1]):
            kk, vv = k[ks[s]:ks[s + 1], h // per], v[ks[s]:ks[s + 1], h // per]
            o, mass, dots, total = ref.attend(q[qs[s]:qs[s + 1], h], kk, vv, ends, scale)
            want[qs[s]:qs[s + 1], h] = o
            top = np.abs(vv).max(initial=0.0)
            bound[qs[s]:qs[s + 1], h] = ref.attention_bound(o, mass, dots, total, top, nk, d)
    return want, bound, used


def run_prompt(amd, q, k, v, qs, ks, causal, scale=None, **kw):
    import torch
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return amd.attention_prompt(to(q), to(k), to(v), to(np.asarray(qs, np.int32)), to(np.asarray(ks, np.int32)),
                                causal=causal, scale=scale, **kw).cpu().numpy()


def starts(lens):
    return [0] + [int(x) for x in np.cumsum(lens)]


PROMPTS = [  # query lengths, key lengths, hq, hk, d, causal
    ([1], [1], 1, 1, 64, True),
    ([1], [1000], 4, 2, 128, True),
    ([37], [37], 8, 2, 256, True),
    ([65], [65], 3, 1, 64, False),
    ([1, 0, 5, 64, 33], [1, 0, 5, 64, 33], 6, 2, 128, True),
    ([130, 7, 256], [131, 300, 256], 4, 4, 64, True),
    ([70, 9], [20, 4], 2, 1, 128, True),          # more queries than keys: the first rows see nothing
    ([12, 40], [0, 3], 2, 2, 64, False),          # a sequence without keys
    ([129, 64], [257, 1], 5, 1, 256, False),
    ([300], [300], 2, 1, 256, True),
    ([513], [700], 2, 2, 128, True),
    # a few rows over many keys, so that two groups of waves share them, and many empty places of a batch
    ([130], [1000], 2, 2, 64, True),
    ([140, 3], [1500, 900], 2, 1, 128, True),
    ([33], [850], 1, 1, 256, False),
    ([300, 70] + [0] * 270 + [513], [300, 75] + [3] + [0] * 269 + [600], 2, 1, 128, True),
    ([257] + [0] * 300 + [40], [257] + [0] * 300 + [1], 1, 1, 64, True),
    ([100, 400] + [0] * 300, [700, 33] + [0] * 300, 1, 1, 256, False),
]


@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"{sum(c[0])}x{sum(c[1])}s{len(c[0])}h{c[2]}-{c[3]}d{c[4]}c{int(c[5])}")
def test_prompt_matches_formula(amd, case):
    lq, lk, hq, hk, d, causal = case
    print("  attention_prompt", [x for x in lq if x], [x for x in lk if x], case[2:], flush=True)
    qs, ks = starts(lq), starts(lk)
    q, k, v = rows(70, qs[-1], hq, d, sigma=2.0), rows(71, max(1, ks[-1]), hk, d), rows(72, max(1, ks[-1]), hk, d)
    want, bound, used = prompt_reference(q, k, v, qs, ks, causal, d ** -0.5)
    got = run_prompt(amd, q, k, v, qs, ks, causal).astype(np.float64)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / np.maximum(bound, 1e-30)).max())


LONG = [  # a few rows over many keys: parts of a walk go to several workgroups
    ([1], [2000], 2, 1, 64, True),
    ([20], [1281], 4, 1, 128, True),
    ([130], [3001], 2, 2, 128, True),
    ([3], [1100], 8, 2, 256, True),
    ([257, 1], [2100, 1600], 1, 1, 256, False),
    ([1000], [1000], 3, 1, 64, True),
    ([700], [1025], 2, 1, 256, True),
    ([0, 5, 40], [2500, 2500, 90], 2, 2, 128, True),
    ([50, 200], [5000, 0], 2, 1, 64, False),
    ([1300, 9], [900, 2400], 1, 1, 128, True),  # the first rows see nothing
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{sum(c[0])}x{sum(c[1])}s{len(c[0])}h{c[2]}-{c[3]}d{c[4]}c{int(c[5])}")
def test_prompt_in_parts(amd, case):
    """against the formula; with a workspace of its own and again the bits are the same"""
    lq, lk, hq, hk, d, causal = case
    print("  attention_prompt in parts", case, flush=True)
    qs, ks = starts(lq), starts(lk)
    nbytes = amd.attention_prompt_workspace_bytes(hq, d, len(lq), qs[-1], ks[-1])
    assert nbytes > 0
    q, k, v = rows(75, qs[-1], hq, d, sigma=2.0), rows(76, ks[-1], hk, d), rows(77, ks[-1], hk, d)
    want, bound, _ = prompt_reference(q, k, v, qs, ks, causal, d ** -0.5)
    got = run_prompt(amd, q, k, v, qs, ks, causal)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    ws = amd.new_workspace(128, 128, 1, nbytes=nbytes)
    ws[-4096:] = 0xff  # what it held does not matter
    assert np.array_equal(got, run_prompt(amd, q, k, v, qs, ks, causal, workspace=ws))
    assert np.array_equal(got, run_prompt(amd, q, k, v, qs, ks, causal))
    with pytest.raises(amd.Exl3Error):
        run_prompt(amd, q, k, v, qs, ks, causal, workspace=ws[:nbytes - 256])


def test_prompt_in_parts_ranges(amd):
    """scores that rise or fall with the keys, so that parts differ by hundreds, and a NaN that only the last rows see"""
    n, pre, d = 70, 1900, 64
    qs, ks = [0, n], [0, n + pre]
    ramp = (np.arange(n + pre) * 0.01).astype(np.float16)
    v = rows(78, n + pre, 1, d)
    for k_of in (ramp, ramp[::-1]):
        q, k = np.ones((n, 1, d), np.float16), np.zeros((n + pre, 1, d), np.float16)
        k[:, 0, :] = k_of[:, None]
        want, bound, _ = prompt_reference(q, k, v, qs, ks, True, 1.0)
        got = run_prompt(amd, q, k, v, qs, ks, True, 1.0).astype(np.float64)
        assert np.all(np.abs(got - want) <= bound)
    clean = run_prompt(amd, q, k, v, qs, ks, True)
    for bad, column in ((np.nan, 5), (np.inf, 60)):
        v2, k2 = v.copy(), k.copy()
        v2[-20, 0, column] = bad  # seen by the last 20 rows
        got = run_prompt(amd, q, k2, v2, qs, ks, True)
        assert np.array_equal(got[:-20], clean[:-20]) and not np.isfinite(got[-20:, 0, column]).any()
        others = np.arange(d) != column
        assert np.array_equal(got[-20:, 0, others], clean[-20:, 0, others])
        k2[-20, 0, column] = np.nan
        got = run_prompt(amd, q, k2, v, qs, ks, True)
        assert np.array_equal(got[:-20], clean[:-20]) and np.isnan(got[-20:]).all()


@pytest.mark.parametrize("sigma,scale", [(30.0, None), (0.01, None), (1.0, -0.2), (1.0, 0.0), (8.0, 1.0)])
def test_prompt_score_ranges(amd, sigma, scale):
    """scores from almost equal to hundreds apart, a negative scale and a zero one"""
    lens, d = [200, 61], 128
    qs = starts(lens)
    q, k, v = rows(80, qs[-1], 2, d, sigma=sigma), rows(81, qs[-1], 1, d), rows(82, qs[-1], 1, d, sigma=0.5)
    v += np.float16(2.0)
    want, bound, _ = prompt_reference(q, k, v, qs, qs, True, d ** -0.5 if scale is None else scale)
    got = run_prompt(amd, q, k, v, qs, qs, True, scale).astype(np.float64)
    assert np.all(np.abs(got - want) <= bound)


def test_prompt_rising_scores(amd):
    """the running maximum grows with every key, and falls with every key"""
    n, d = 333, 64
    ramp = (np.arange(n) * 0.06).astype(np.float16)
    for k_of in (ramp, ramp[::-1]):
        q, k, v = np.ones((n, 1, d), np.float16), np.zeros((n, 1, d), np.float16), rows(84, n, 1, d)
        k[:, 0, :] = k_of[:, None]
        want, bound, _ = prompt_reference(q, k, v, [0, n], [0, n], True, 1.0)
        got = run_prompt(amd, q, k, v, [0, n], [0, n], True, 1.0).astype(np.float64)
        assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("poison", [np.nan, np.inf, -np.inf, 65504.0])
def test_prompt_masked_places_do_not_reach_a_row(amd, poison):
    """keys and values that a row does not see (after its end, of other sequences, of none) hold anything"""
    import torch
    lens, d = [50, 20], 128
    qs = starts(lens)
    q, k, v = rows(90, 80, 2, d), rows(91, 80, 1, d), rows(92, 80, 1, d)
    clean = run_prompt(amd, q, k, v, qs, qs, True)
    for at in (49, 69, 75):  # the last key of each sequence, a row of no sequence
        kk, vv = k.copy(), v.copy()
        kk[at], vv[at] = poison, poison
        got = run_prompt(amd, q, kk, vv, qs, qs, True, out=torch.zeros((80, 2, d), dtype=torch.float16, device="cuda"))
        keep = np.ones(80, bool)
        keep[at] = keep[70:] = False
        assert np.array_equal(got[keep], clean[keep]), at


def test_prompt_leaves_other_rows_and_views(amd):
    """head-major, sliced and unaligned views; rows of no sequence keep what they held"""
    import torch
    lens, hq, hk, d = [40, 25], 4, 2, 64
    qs = starts(lens)
    n = qs[-1] + 6
    q, k, v = rows(95, n, hq, d), rows(96, n, hk, d), rows(97, n, hk, d)
    want = run_prompt(amd, q, k, v, qs, qs, True)[:qs[-1]]
    width = (hq + 2 * hk) * d + 3
    buf = torch.zeros(n * width + 1, dtype=torch.float16, device="cuda")
    view = buf[1:].view(n, width)
    parts = []
    at = 0
    for a, h in ((q, hq), (k, hk), (v, hk)):
        piece = view[:, at:at + h * d].unflatten(1, (h, d))
        piece.copy_(torch.from_numpy(a))
        parts.append(piece)
        at += h * d
    st = torch.tensor(qs, dtype=torch.int32, device="cuda")
    out = torch.full((hq, n, d), 9.0, dtype=torch.float16, device="cuda")
    amd.attention_prompt(*parts, st, out=out.transpose(0, 1))
    got = out.transpose(0, 1).cpu().numpy()
    assert np.array_equal(got[:qs[-1]], want) and np.all(got[qs[-1]:] == 9.0)


def test_prompt_starts_beyond_the_rows(amd):
    """starts that do not fit the views: nothing outside them is read or written"""
    import torch
    d = 64
    q = rows(98, 30, 1, d)
    for qs, ks in (([0, 30], [0, 4000]), ([0, 4000], [0, 30]), ([-5, 30], [-9, 30]), ([20, 10], [0, 30]),
                   ([0, 30], [25, 5])):
        out = run_prompt(amd, q, q, q, qs, ks, True, out=torch.zeros((30, 1, d), dtype=torch.float16, device="cuda"))
        assert out.shape == (30, 1, d)


# ------------------------------------------------------------------ the cache
def make_cache(amd, lens, heads, d, bits, p, width=None, seed=100, spare=3):
    """(pages, table, rotated keys and values of each sequence) with random rows in shuffled pages; the rest of the
    pages is filled with bytes that read as NaN and infinities"""
    import torch
    need = [-(-n // p) for n in lens]
    width = max([1] + need) if width is None else width
    count = sum(need) + spare
    size = amd.kv_page_bytes(heads, d, bits, p)
    pages = np.full((count, size), 0xFF, np.uint8)
    order = np.argsort(synth.splitmix64(seed, count))
    table = np.full((len(lens), width), int(order[-1]), np.int32)  # unused places point at a page of NaN
    kept, at = [], 0
    for s, n in enumerate(lens):
        k, v = rows(seed + 2 * s, max(n, 1), heads, d), rows(seed + 2 * s + 1, max(n, 1), heads, d, sigma=0.6)
        (kc, ks), (vc, vs) = ref.quantise(k, bits), ref.quantise(v, bits)
        for j in range(need[s]):
            page = int(order[at + j])
            table[s, j] = page
            parts = [a.copy() for a in ref.page_parts(pages[page], bits, heads, d, p)]
            m = min(p, n - j * p)
            for part, src in zip(parts, (kc, vc, ks, vs)):
                part[:, :m] = src[j * p:j * p + m].transpose(1, 0, 2)
            pages[page] = ref.pack_page(*parts, bits)
        kept.append((ref.values(kc, ks, bits)[:n], ref.values(vc, vs, bits)[:n]))
        at += need[s]
    return torch.from_numpy(pages).cuda(), torch.from_numpy(table).cuda(), kept


def cached_reference(q, kept, q_len, heads, scale):
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    per, d = q.shape[1] // heads, q.shape[2]
    qr = ref.rotate(q.astype(np.float64))
    for s, (k, v) in enumerate(kept):
        n = len(k)
        ends = n - (q_len - 1 - np.arange(q_len))
        for h in range(q.shape[1]):
            at = slice(s * q_len, (s + 1) * q_len)
            kk, vv = k[:, h // per], v[:, h // per]
            o, mass, dots, total = ref.attend(qr[at, h], kk, vv, ends, scale)
            # the bound of the rotated row; rotating back sums 32 elements of it with +-1/sqrt(32), in binary32
            b = ref.attention_bound(o, mass, dots, total, np.abs(vv).max(initial=0.0), n, d)
            b = b.reshape(q_len, -1, 32)
            o32 = np.abs(o).reshape(q_len, -1, 32)
            both = (b.sum(-1, keepdims=True) + 6 * 2.0 ** -24 * o32.sum(-1, keepdims=True)) / np.sqrt(32)
            want[at, h] = ref.rotate(o)
            bound[at, h] = np.broadcast_to(both, b.shape).reshape(q_len, d) + ref.U16 * np.abs(want[at, h]) + 2.0 ** -25
    return want, bound


def run_cached(amd, q, pages, table, lens, heads, bits, p, q_len, **kw):
    import torch
    return amd.attention_cached(torch.from_numpy(q).cuda(), pages, table,
                                torch.tensor(lens, dtype=torch.int32, device="cuda"), heads, bits=bits, page_tokens=p,
                                q_len=q_len, **kw).cpu().numpy()


CACHED = [  # lengths, hq, hk, d, bits, page, q_len
    ([1], 1, 1, 64, 4, 16, 1),
    ([17], 8, 2, 256, 4, 16, 1),
    ([1000], 8, 2, 256, 4, 16, 1),
    ([31, 0, 33, 400], 4, 4, 128, 4, 32, 1),
    ([500, 64, 3], 12, 4, 64, 8, 64, 4),
    ([700, 2], 5, 1, 128, 8, 48, 3),           # a sequence shorter than its new tokens: rows that see nothing
    ([129, 255, 1000, 5, 77], 6, 2, 128, 4, 256, 1),
    ([333], 40, 1, 64, 4, 16, 7),              # more rows per kv head than one tile
    ([260, 90], 16, 2, 256, 8, 16, 2),
    ([2500], 3, 3, 128, 4, 80, 1),
    ([64] * 20, 2, 1, 64, 4, 16, 1),
]


@pytest.mark.parametrize("case", CACHED, ids=str)
def test_cached_matches_formula(amd, case):
    lens, hq, hk, d, bits, p, q_len = case
    print("  attention_cached", case, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(120, len(lens) * q_len, hq, d, sigma=2.0)
    want, bound = cached_reference(q, kept, q_len, hk, d ** -0.5)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len).astype(np.float64)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / np.maximum(bound, 1e-30)).max())


@pytest.mark.parametrize("q_len,hq,hk,d,bits", [(7, 16, 2, 128, 8), (3, 24, 3, 64, 4), (5, 7, 1, 256, 4), (17, 2, 1, 128, 4)])
def test_cached_last_row_tile_is_smaller(amd, q_len, hq, hk, d, bits):
    """rows that are no multiple of 16, over sequences that several workgroups share"""
    lens, p = [4100, 900, 0, 2600, 17], 64
    print("  attention_cached", q_len, hq, hk, d, bits, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(140, len(lens) * q_len, hq, d, sigma=2.0)
    want, bound = cached_reference(q, kept, q_len, hk, d ** -0.5)
    for _ in range(2):
        got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len).astype(np.float64)
        assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("q_len,hq,hk,d,bits", [(1, 4, 1, 256, 4), (3, 8, 1, 256, 8), (8, 8, 2, 128, 4), (9, 16, 1, 64, 8)])
def test_cached_joined_apart(amd, q_len, hq, hk, d, bits):
    """sequences long enough that a second kernel joins their parts, beside short and empty ones; a NaN token"""
    import torch
    lens, p = [9000, 0, 300, 5001, 1], 64
    print("  attention_cached", q_len, hq, hk, d, bits, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(150, len(lens) * q_len, hq, d, sigma=2.0)
    want, bound = cached_reference(q, kept, q_len, hk, d ** -0.5)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len)
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    assert np.array_equal(got, run_cached(amd, q, pages, table, lens, hk, bits, p, q_len))
    slot = torch.tensor([int(table[3, 40]) * p + 7], device="cuda")
    k, v = amd.kv_cache_read(pages, slot, hk, d, bits=bits, page_tokens=p)
    k[:] = float("nan")
    amd.kv_cache_write(pages, k, v, slot, bits=bits, page_tokens=p)
    bad = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len)
    assert np.isnan(bad[3 * q_len:4 * q_len]).all()
    others = np.r_[0:3 * q_len, 4 * q_len:5 * q_len]
    assert np.array_equal(bad[others], got[others])


@pytest.mark.parametrize("bits", [4, 8])
def test_cached_long(amd, bits):
    """one long sequence beside short ones; the table is wider than any of them"""
    lens, hq, hk, d, p = [9001, 3, 700], 4, 2, 128, 64
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p, width=160)
    q = rows(130, 3, hq, d, sigma=3.0)
    want, bound = cached_reference(q, kept, 1, hk, 0.11)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, 1, scale=0.11).astype(np.float64)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("sigma,scale", [(30.0, None), (0.01, None), (1.0, -0.2), (1.0, 0.0), (8.0, 1.0)])
def test_cached_score_ranges(amd, sigma, scale):
    """scores from almost equal to hundreds apart, a negative scale and a zero one"""
    lens, hq, hk, d, bits, p = [300, 45], 4, 2, 128, 4, 16
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    q = rows(170, 2 * 3, hq, d, sigma=sigma)
    want, bound = cached_reference(q, kept, 3, hk, d ** -0.5 if scale is None else scale)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, 3, scale=scale).astype(np.float64)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("bits,d", [(4, 64), (4, 128), (4, 256), (8, 128)])
def test_cached_non_finite_tokens(amd, bits, d):
    """a new token whose keys or values are not finite reaches the rows that see it, and only those"""
    lens, hq, hk, p, q_len = [70, 129], 4, 2, 16, 4
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    import torch
    q = rows(180, 2 * q_len, hq, d)
    clean = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len)
    for which in ("k", "v"):
        for back in (0, 1, 3):  # tokens from the end of sequence 1: token j of q_len sees it when j >= q_len - 1 - back
            dirty = pages.clone()
            at = lens[1] - 1 - back
            slot = int(table[1, at // p]) * p + at % p
            k, v = amd.kv_cache_read(pages, torch.tensor([slot], device="cuda"), hk, d, bits=bits, page_tokens=p)
            (k if which == "k" else v)[0, 1, 5] = float("nan")
            amd.kv_cache_write(dirty, k, v, torch.tensor([slot], device="cuda"), bits=bits, page_tokens=p)
            got = run_cached(amd, q, dirty, table, lens, hk, bits, p, q_len)
            per = hq // hk
            assert np.array_equal(got[:q_len], clean[:q_len])
            rest = got[q_len:]
            sees = np.arange(q_len) >= q_len - 1 - back
            bad = np.isnan(rest[:, per:])  # the q heads of kv head 1
            if which == "k":
                assert bad[sees].all()
            else:
                assert bad[sees][:, :, :32].all() and not bad[sees][:, :, 32:].any()
            assert not np.isnan(rest[~sees]).any() and not np.isnan(rest[:, :per]).any()
            assert np.array_equal(rest[~sees][:, per:], clean[q_len:][~sees][:, per:])


def test_cached_workspaces_streams_and_repeats(amd):
    """the caller's workspace (which mul_mat may share), the internal one, another stream: the same bits"""
    import torch
    lens, hq, hk, d, bits, p = [800, 90, 0], 8, 2, 128, 4, 16
    pages, table, _ = make_cache(amd, lens, hk, d, bits, p)
    q = rows(140, 3, hq, d)
    first = run_cached(amd, q, pages, table, lens, hk, bits, p, 1)
    nbytes = amd.attention_cached_workspace_bytes(hq, hk, d, 3)
    ws = amd.new_workspace(128, 128, 1, nbytes=nbytes)
    for _ in range(3):
        assert np.array_equal(run_cached(amd, q, pages, table, lens, hk, bits, p, 1, workspace=ws), first)
    assert not amd.workspace_faulted(ws)
    with pytest.raises(amd.Exl3Error) as e:
        run_cached(amd, q, pages, table, lens, hk, bits, p, 1, workspace=ws[:nbytes - 1])
    assert e.value.status == amd.WORKSPACE_TOO_SMALL
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run_cached(amd, q, pages, table, lens, hk, bits, p, 1)
    assert np.array_equal(other, first)


def test_cached_bad_pages_and_lengths(amd):
    """an entry outside the cache makes its sequence's rows NaN and no other's; lengths are held to the table"""
    import torch
    lens, hq, hk, d, bits, p = [100, 100, 40], 4, 2, 64, 4, 16
    pages, table, _ = make_cache(amd, lens, hk, d, bits, p)
    q = rows(150, 3, hq, d)
    clean = run_cached(amd, q, pages, table, lens, hk, bits, p, 1)
    for entry in (-1, pages.shape[0], 2 ** 31 - 1, -(2 ** 31)):
        t = table.clone()
        t[1, 2] = entry
        got = run_cached(amd, q, pages, t, lens, hk, bits, p, 1)
        assert np.isnan(got[1]).all() and np.array_equal(got[[0, 2]], clean[[0, 2]])
        t = table.clone()
        t[2, 4:] = entry  # places that nothing reads
        assert np.array_equal(run_cached(amd, q, pages, t, lens, hk, bits, p, 1), clean)
    capped = run_cached(amd, q, pages, table, [2 ** 31 - 1, 100, -7], hk, bits, p, 1)
    full = run_cached(amd, q, pages, table, [table.shape[1] * p, 100, 0], hk, bits, p, 1)
    assert np.array_equal(capped, full, equal_nan=True) and np.all(capped[2] == 0)


def test_cached_views_and_far_pages(amd):
    """head-major and unaligned rows, and a cache beyond 4 GiB"""
    import torch
    lens, hq, hk, d, bits, p = [75], 4, 2, 64, 4, 16
    pages, table, _ = make_cache(amd, lens, hk, d, bits, p)
    q = rows(160, 1, hq, d)
    want = run_cached(amd, q, pages, table, lens, hk, bits, p, 1)
    far = torch.zeros(((1 << 32) // pages.shape[1] + 40, pages.shape[1]), dtype=torch.uint8, device="cuda")
    off = far.shape[0] - pages.shape[0]
    far[off:] = pages
    buf = torch.zeros(hq * (d + 3) + 1, dtype=torch.float16, device="cuda")
    qv = buf[1:].view(1, hq, d + 3)[:, :, :d]
    qv.copy_(torch.from_numpy(q))
    out = torch.zeros_like(buf)[1:].view(1, hq, d + 3)[:, :, :d]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    amd.attention_cached(qv, far, table + off, ln, hk, bits=bits, page_tokens=p, out=out)
    assert np.array_equal(out.cpu().numpy(), want)


# ------------------------------------------------------------------ together
def test_block_in_a_captured_graph(amd):
    """norm and positions, cache write, attention over cache and prompt in one HIP graph: each replay equals the
    eager calls, with eager work in between, also after the inputs have changed"""
    import torch
    hq, hk, d, bits, p, n = 8, 2, 128, 4, 16, 300
    g = torch.Generator(device="cuda").manual_seed(5)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731
    qkv = draw(n, (hq + 2 * hk), d)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    f = torch.from_numpy((1e4 ** (-np.arange(0, d, 2) / d)).astype(np.float32)).cuda()
    w = torch.ones(d, device="cuda")
    pages = amd.new_kv_cache(20, hk, d, bits, p)
    slots = torch.arange(n, device="cuda")
    table = torch.arange(19, dtype=torch.int32, device="cuda")[None].contiguous()
    lens, starts_ = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([n], [0, n]))
    ws = amd.new_workspace(128, 128, 1, nbytes=amd.attention_cached_workspace_bytes(hq, hk, d, 1))

    def step():
        q, k = amd.qk_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hk], pos, f, w, w)
        v = qkv[:, hq + hk:]
        amd.kv_cache_write(pages, k, v, slots, bits=bits, page_tokens=p)
        rk, rv = amd.kv_cache_read(pages, slots, hk, d, bits=bits, page_tokens=p)
        a = amd.attention_prompt(q, rk, rv, starts_)
        b = amd.attention_cached(q[-1:], pages, table, lens, hk, bits=bits, page_tokens=p, workspace=ws)
        return a, b

    def eager():
        out = tuple(t.clone() for t in step())
        torch.cuda.synchronize()
        return out

    first = eager()
    # the last row of the prompt and the cached step see the same keys and values
    assert (first[0][-1].float() - first[1][0].float()).abs().max() < 0.01
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a, b = step()
    for r in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, first[0]) and torch.equal(b, first[1]), r
        if r == 1:
            qkv.copy_(draw(n, hq + 2 * hk, d))
        first = eager()
