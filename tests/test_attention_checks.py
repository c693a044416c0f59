"""Arguments of the attention block's entry points that have to be refused on the host: scales that are not finite."""
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
