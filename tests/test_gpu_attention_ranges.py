"""Attention over the cache with queries and cached groups near the ends of fp16, against the formula in 64 bits
within attention_ref.attention_bound: a finite row gives finite, right results whatever its rotation by H32 makes of
it, which is up to sqrt(32) times its largest element."""
import numpy as np
import pytest

import attention_ref as ref
from test_gpu_attention import cached_reference, make_cache, rows, run_cached

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,bits,lens,q_len", [(64, 4, [90, 17], 3), (128, 8, [700], 2), (256, 4, [300, 5000], 1)])
@pytest.mark.parametrize("size", [11000.0, 12000.0, 65504.0])
def test_queries_whose_rotation_passes_fp16(amd, d, bits, lens, q_len, size):
    """32 equal elements of 12,000 rotate to 67,882; the other rows keep their bits"""
    hq, hk, p = 4, 2, 16
    print("  attention_cached", d, bits, lens, q_len, size, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    plain = rows(200, len(lens) * q_len, hq, d, sigma=2.0)
    q = plain.copy()
    q[0, 1, :32] = size
    q[-1, 3, 32:64] = -size
    q[-1, 2] = np.where(rows(201, d) > 0, size, -size)
    scale = 1.0 / size
    want, bound = cached_reference(q, kept, q_len, hk, scale)
    got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len, scale=scale)
    assert np.isfinite(got).all()
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    same = np.ones(q.shape[:2], bool)
    same[0, 1] = same[-1, 2] = same[-1, 3] = False
    assert np.array_equal(got[same], run_cached(amd, plain, pages, table, lens, hk, bits, p, q_len, scale=scale)[same])


LARGE = [  # bits, d, lengths, q_len, size of the keys, size of the values
    (4, 64, [33, 90], 4, 12000.0, 12000.0),
    (8, 64, [90], 4, 65504.0, 12000.0),
    (4, 128, [700, 130], 3, 90000.0, 30000.0),
    (8, 128, [2600], 1, 1.3e6, 30000.0),
    (4, 256, [40, 4100], 4, 12000.0, 40000.0),
    (8, 256, [129], 2, 12000.0, 12000.0),
]


@pytest.mark.parametrize("case", LARGE, ids=str)
def test_cached_groups_whose_products_pass_fp16(amd, case):
    """32 equal elements of 12,000 have a finite scale, but scale * code is 68,000: tokens with such groups of keys and
    values, among them new ones that the first rows do not see, beside ordinary tokens of the same tile"""
    import torch
    bits, d, lens, q_len, k_size, v_size = case
    hq, hk, p, n = 4, 2, 16, lens[-1]
    print("  attention_cached", case, flush=True)
    pages, table, kept = make_cache(amd, lens, hk, d, bits, p)
    where = [3, n // 2, n - 2, n - 1]
    k, v = rows(210, 4, hk, d, sigma=0.8).astype(np.float32), rows(211, 4, hk, d, sigma=0.6).astype(np.float32)
    for i in range(4):  # the second head's last group and the first head's first one
        k[i, 0, :32] = v[i, 1, -32:] = 1.0 if i % 2 else -1.0
        k[i, 0, :32] *= k_size
        v[i, 1, -32:] *= v_size
    v[:, 0, :32] = np.abs(v[:, 0, :32]) * v_size / 4
    slots = torch.tensor([int(table[-1, t // p]) * p + t % p for t in where], device="cuda")
    amd.kv_cache_write(pages, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), slots, bits=bits, page_tokens=p)
    for rows_of, x in zip(kept[-1], (k, v)):
        code, s = ref.quantise(x, bits)
        assert np.isfinite(s).all()
        rows_of[where] = ref.values(code, s, bits)
    assert max(np.abs(a[where]).max() for a in kept[-1]) > 65504
    q = rows(213, len(lens) * q_len, hq, d, sigma=2.0)
    for scale in (1.0 / k_size, d ** -0.5):  # the large keys beside the others, and far ahead of or behind them
        want, bound = cached_reference(q, kept, q_len, hk, scale)
        got = run_cached(amd, q, pages, table, lens, hk, bits, p, q_len, scale=scale)
        assert np.isfinite(got).all()
        assert np.all(np.abs(got.astype(np.float64) - want) <= bound)


@pytest.mark.parametrize("d,n", [(64, 53000), (128, 14000), (256, 6000)])
def test_joined_apart_with_odd_rows(amd, d, n):
    """five rows of each of two kv heads over one long sequence, whose parts a second kernel joins"""
    print("  attention_cached", d, n, flush=True)
    pages, table, kept = make_cache(amd, [n], 2, d, 4, 64)
    q = rows(220, 1, 10, d, sigma=2.0)
    want, bound = cached_reference(q, kept, 1, 2, d ** -0.5)
    got = run_cached(amd, q, pages, table, [n], 2, 4, 64, 1)
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
