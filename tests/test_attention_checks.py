"""Arguments of the attention block's entry points that have to be refused on the host: scales that are not finite, views
beyond any address space."""
import ctypes

import pytest

import conftest

INVAL = 1
P, Q = 0x100000, 0x200000  # stand-ins for device addresses: no refused call reaches the device


@pytest.fixture(scope="module")
def L():
    return conftest.load_amd().lib()


def view(data=P, heads=2, token=256, head=128):
    return ctypes.byref(conftest.load_amd().HeadView(data, heads, token, head))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_scale_is_finite(L, scale):
    """a NaN would pass the bound from below that the exponent's factor has, and every key weigh the same"""
    assert L.exl3_hip_attention_cached(view(), view(Q), 128, P, 4, 4, 16, 1, P, 9, P, 2, 1, scale, None, 0, None) == INVAL
    assert L.exl3_hip_attention_prompt(view(), view(heads=1), view(heads=1), view(Q), 128, P, P, 1, 3, 3, scale, 1, None,
                                       0, None) == INVAL


WRAPS = (2, 1 << 35, 1 << 36, (1 << 29) + 1)  # heads, token stride, head stride, tokens: (tokens - 1) * stride is 2^64


def test_views_whose_offsets_wrap(L):
    """the overlap test's products wrap in 64 bits: token 2 of head 0 is token 0 of head 1, and passed as disjoint"""
    heads, token, head, tokens = WRAPS
    out = view(Q, heads, token, head)
    one = view(heads=heads)
    assert L.exl3_hip_qk_norm_rope(one, None, 1, tokens, 128, None, None, 0.0, None, None, 0, 0, 1.0, out, None, 1,
                                   None) == INVAL
    assert L.exl3_hip_kv_cache_read(P, 4, 4, 16, 128, P, tokens, out, out, 1, None, None) == INVAL
    assert L.exl3_hip_attention_prompt(one, view(heads=1), view(heads=1), out, 128, P, P, 1, tokens, 3, 0.1, 1, None, 0,
                                       None) == INVAL
    # and rows that are only read, from 2^48 elements on
    for x, n in ((view(P, 2, 1 << 40, 128), 1 << 9), (view(P, 300, 256, 1 << 40), 1)):
        assert L.exl3_hip_qk_norm_rope(x, None, 1, n, 128, None, None, 0.0, None, None, 0, 0, 1.0,
                                       view(Q, 2 if n > 1 else 300), None, 1, None) == INVAL


def test_partials_are_aligned(L):
    """the partials of every (kv head, row tile) are read 16 bytes at a time: their sizes are whole 256 bytes, for odd rows,
    tiles and partial counts too"""
    prefix = (16 << 20) + 256  # the exchange and the status block
    for hq, hk, d, seqs, q_len, tiles in ((10, 2, 128, 1, 1, 2), (3, 1, 64, 7, 1, 1), (9, 3, 256, 5, 3, 3), (7, 1, 64, 2, 5, 3)):
        need = L.exl3_hip_attention_cached_workspace_bytes(hq, hk, d, seqs, q_len)
        assert need > prefix and (need - prefix) % (256 * tiles) == 0, (hq, hk, d, seqs, q_len)
