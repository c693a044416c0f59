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
