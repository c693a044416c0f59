"""exl3_hip_short_conv against the formula in 64 bits."""
import numpy as np
import pytest

import linear_attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def rows(seed, shape, dtype="float32", sigma=1.0):
    return synth.normal(seed, int(np.prod(shape)), sigma).reshape(shape).astype(dtype)


def cuda(a):
    import torch
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check(got, want, bound, dtype):
    got = got.cpu().numpy()
    assert str(got.dtype) == dtype
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.nan_to_num(np.abs(got.astype(np.float64) - want))
    assert np.all(err <= np.nan_to_num(bound + ref.rounded(np.abs(want) + bound, dtype))), float(np.max(err))


def starts_of(lens):
    import torch
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def run(amd, lens, channels, width, x, y, silu, bias, states, sin, sout, packed=True, behind=2, seed=1):
    import torch
    n = sum(lens)
    a = rows(seed, (n + behind, channels), x)
    a[n:] = np.nan
    w, b = rows(seed + 1, (channels, width), sigma=0.5), rows(seed + 2, (channels,)) if bias else None
    pool = None if states is None else cuda(states)
    out = torch.full((n + behind, channels), 5.0, dtype=getattr(torch, y), device="cuda")
    kw = dict(starts=starts_of(lens)) if packed else dict(sequences=len(lens))
    assert packed or behind == 0
    amd.short_conv(cuda(a), cuda(w), bias=cuda(b), silu=silu, states=pool, slots_in=cuda(sin), slots_out=cuda(sout),
                   out=out, **kw)
    want, after, bound = ref.short_conv(a[:n].astype(np.float64), w.astype(np.float64),
                                        None if b is None else b.astype(np.float64), silu, lens,
                                        None if states is None else states.astype(np.float64), sin, sout)
    check(out[:n], want, bound, y)
    assert bool((out[n:] == 5).all())
    if states is not None:
        assert np.array_equal(pool.cpu().numpy(), after.astype(states.dtype), equal_nan=True)


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [1, 24, 131, 256, 2048, 2056])
@pytest.mark.parametrize("x,y", [("float16", "float16"), ("float32", "float16"), ("float16", "float32"),
                                 ("float32", "float32")])
def test_packed_rows(amd, width, channels, x, y):
    """sequences of none, one, two, .. rows around the tiles' ends, some from states and some from zeros"""
    lens = [0, 1, 2, 3, 4, 5, 31, 32, 33, 0, 70, 1]
    m = len(lens)
    states = rows(9, (m + 2, width - 1, channels), x)
    order = np.random.default_rng(3).permutation(m + 2)[:m].astype(np.int32)
    sin = order.copy()
    sin[[3, 7]] = -1
    run(amd, lens, channels, width, x, y, channels != 24, channels != 256, states, sin, order)


@pytest.mark.parametrize("lens", [[1] * 9, [2] * 3, [3], [0, 0], [8] * 70, [700], [4096]])
def test_as_many_rows_each(amd, lens):
    states = rows(9, (len(lens), 3, 264), "float16")
    slots = np.random.default_rng(4).permutation(len(lens)).astype(np.int32)
    run(amd, lens, 264, 4, "float16", "float16", True, False, states, slots, slots, packed=False, behind=0)


def test_without_states(amd):
    run(amd, [5, 0, 40], 72, 4, "float32", "float32", True, True, None, None, None)


@pytest.mark.parametrize("channels", [16, 17])
def test_slots_that_are_none_or_beyond_the_pool(amd, channels):
    states = rows(9, (4, 3, channels))
    run(amd, [1, 2, 6, 0, 7], channels, 4, "float32", "float32", False, False, states,
        np.array([4, 1 << 30, 9, 2, -5], np.int32), np.array([0, 1, 4, 3, -2], np.int32))


def test_a_state_read_by_two_and_moved(amd):
    states = rows(9, (4, 3, 64))
    run(amd, [1, 9, 0], 64, 4, "float32", "float32", True, False, states, np.array([1, 1, 1], np.int32),
        np.array([0, 2, 3], np.int32))


@pytest.mark.parametrize("cuts", [[10], [1, 2, 3, 4], [1] * 10, [4, 0, 6]])
def test_pieces_are_the_whole(amd, cuts):
    """a sequence in pieces over its state gives the bits of the sequence at once"""
    import torch
    x, w = cuda(rows(1, (10, 40), "float16")), cuda(rows(2, (40, 4)))
    whole = amd.short_conv(x, w, starts=starts_of([10]))
    states, slot = amd.new_conv_states(1, 40), torch.zeros(1, dtype=torch.int32, device="cuda")
    got, at = [], 0
    for n in cuts:
        got.append(amd.short_conv(x[at:at + n], w, states=states, slots_in=slot, slots_out=slot))
        at += n
    assert torch.equal(torch.cat(got), whole) and torch.equal(states[0], x[-3:])


def test_strided_rows(amd):
    import torch
    wide = cuda(rows(1, (37, 80), "float16"))
    w = cuda(rows(2, (40, 4)))
    for off in (8, 3):
        x = wide[:, off:off + 40]
        out = torch.zeros(37, 48, dtype=torch.float16, device="cuda")
        amd.short_conv(x, w, out=out[:, 2:42])
        assert torch.equal(out[:, 2:42], amd.short_conv(x.contiguous(), w))
        assert bool((out[:, :2] == 0).all() and (out[:, 42:] == 0).all())


def test_starts_that_are_no_packing(amd):
    """no row outside the views is read or written; the rows of the good sequences are theirs"""
    import torch
    x, w = cuda(rows(1, (20, 64), "float16")), cuda(rows(2, (64, 4)))
    starts = torch.tensor([-5, 4, 2, 9, 100], dtype=torch.int32, device="cuda")
    got = amd.short_conv(x, w, starts=starts)
    assert torch.equal(got[9:], amd.short_conv(x[9:], w)) and torch.equal(got[:4][:2], amd.short_conv(x[:2], w))
