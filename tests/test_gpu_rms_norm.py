"""exl3_hip_rms_norm against the formula in 64 bits."""
import numpy as np
import pytest

import linear_attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def rows(seed, shape, dtype, sigma=1.0):
    return synth.normal(seed, int(np.prod(shape)), sigma).reshape(shape).astype(dtype)


def cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def check(got, want, bound, dtype):
    got = got.cpu().numpy()
    assert str(got.dtype) == dtype
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= bound + ref.rounded(np.abs(want) + bound, dtype)), float(np.max(err))


WIDTHS = [1, 7, 8, 40, 64, 128, 136, 256, 512, 520, 1531, 2048, 4096, 8192, 8200, 16384, 16392, 65536]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("x,r,y", [("float16", None, "float16"), ("float32", "float32", "float16"),
                                   ("float16", "float32", "float32"), ("float32", "float16", "float32")])
def test_widths_and_types(amd, width, x, r, y):
    import torch
    n = 5 if width > 4096 else 67
    a, w = rows(1, (n, width), x, 3.0), 1 + 0.2 * rows(2, (width,), "float32")
    a[0] = 0
    res = None if r is None else rows(3, (n, width), r)
    out = amd.rms_norm(cuda(a), cuda(w), residual=None if r is None else cuda(res), eps=1e-5,
                       out_dtype=getattr(torch, y))
    want, h, bound = ref.rms_norm(a.astype(np.float64), w.astype(np.float64), float(np.float32(1e-5)),
                                  None if r is None else res.astype(np.float64))
    if r is not None:
        out, kept = out
        check(kept, h, ref.E32 * np.abs(h), r)
    check(out, want, bound, y)


@pytest.mark.parametrize("x", ["float16", "float32"])
@pytest.mark.parametrize("heads,width", [(16, 128), (3, 64), (2, 256), (5, 72), (1, 2048), (7, 33)])
def test_gated_heads_of_a_wider_row(amd, x, heads, width):
    """heads are slices of rows that hold more than them; the gate another slice"""
    import torch
    n = 41
    wide = rows(4, (n, 2 * heads * width + 24), x)
    t = cuda(wide)
    a, z = t[:, 8:8 + heads * width].view(n, heads, width), t[:, 16 + heads * width:16 + 2 * heads * width]
    z = z.view(n, heads, width)
    w = 1 + 0.2 * rows(5, (width,), "float32")
    out = amd.rms_norm(a, cuda(w), gate=z, out_dtype=torch.float16)
    want, _, bound = ref.rms_norm(a.cpu().numpy().astype(np.float64), w.astype(np.float64), float(np.float32(1e-6)),
                                  gate=z.cpu().numpy().astype(np.float64))
    check(out, want, bound, "float16")


@pytest.mark.parametrize("width", [128, 131, 2048])
def test_in_place_and_rows_left_alone(amd, width):
    import torch
    n = 9
    a, r = rows(6, (n, width), "float32"), rows(7, (n, width), "float32")
    w = rows(8, (width,), "float32")
    want = amd.rms_norm(cuda(a), cuda(w), residual=cuda(r))
    buf = torch.full((n + 2, width + 8), 7.0, device="cuda")
    buf[1:-1, :width] = cuda(a)
    x, res = buf[1:-1, :width], cuda(r)
    out, kept = amd.rms_norm(x, cuda(w), residual=res, out=x, residual_out=res)
    assert kept is res or kept.data_ptr() == res.data_ptr()
    assert torch.equal(out, want[0]) and torch.equal(res, want[1])
    assert bool((buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, width:] == 7).all())


def test_without_weight_and_of_no_rows(amd):
    import torch
    a = rows(9, (3, 96), "float16")
    want, _, bound = ref.rms_norm(a.astype(np.float64), None, 0.0)
    check(amd.rms_norm(cuda(a), eps=0.0), want, bound, "float16")
    assert amd.rms_norm(torch.empty(0, 96, device="cuda"), None).shape == (0, 96)


@pytest.mark.parametrize("scale", [1e-30, 1e-19, 1e-3, 1e4, 1e18])
def test_sizes_of_the_elements(amd, scale):
    """squares of 1e-30 vanish in 32 bits: eps carries those rows; 1e18 leaves room for the sum of 256 squares"""
    import torch
    a = (rows(10, (4, 256), "float32").astype(np.float64) * scale).astype(np.float32)
    want, _, bound = ref.rms_norm(a.astype(np.float64), None, float(np.float32(1e-6)))
    check(amd.rms_norm(cuda(a)), want, bound, "float32")


def test_nan_and_infinity_stay_in_their_row(amd):
    import torch
    a = rows(11, (4, 2048), "float32")
    clean = amd.rms_norm(cuda(a)).cpu()
    a[1, 5], a[2, 2047] = np.nan, np.inf
    got = amd.rms_norm(cuda(a)).cpu()
    assert torch.equal(got[[0, 3]], clean[[0, 3]]) and bool(torch.isnan(got[1]).all())
    assert bool((got[2, :2047] == 0).all()) and bool(torch.isnan(got[2, 2047]))
