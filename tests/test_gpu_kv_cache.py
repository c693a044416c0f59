"""The quantised cache: page bytes bit for bit against a restatement of the format in binary32 numpy, rows read
back against its values in 64 bits.  Reading sums 32 values in five binary32 stages and scales them: within 6 *
2^-24 of the sum of their magnitudes / sqrt(32); then one rounding to the output type."""
import numpy as np
import pytest

import attention_ref as ref
import synth

pytestmark = pytest.mark.gpu


def rows(seed, tokens, heads, d, dtype, sigma=1.0):
    x = synth.normal(seed, tokens * heads * d, sigma).reshape(tokens, heads, d)
    x *= np.exp(synth.normal(seed + 1, heads * d, 0.7)).reshape(heads, d)
    return x.astype(np.float16 if dtype == "f16" else np.float32)


def expected_pages(before, k, v, slots, bits, p):
    heads, d = k.shape[1:]
    kc, ks = ref.quantise(k, bits)
    vc, vs = ref.quantise(v, bits)
    out = before.copy()
    for page in sorted({int(s) // p for s in slots if 0 <= s < len(out) * p}):
        parts = [a.copy() for a in ref.page_parts(out[page], bits, heads, d, p)]
        for t, s in enumerate(slots):
            if s >= 0 and int(s) // p == page:
                at = int(s) % p
                parts[0][:, at], parts[1][:, at], parts[2][:, at], parts[3][:, at] = kc[t], vc[t], ks[t], vs[t]
        out[page] = ref.pack_page(*parts, bits)
    return out


def read_bound(code, scale, bits):
    mass = np.abs(ref.values(code, scale, bits)).reshape(*scale.shape, 32).sum(-1, keepdims=True) / np.sqrt(32)
    return 6 * 2.0 ** -24 * np.broadcast_to(mass, (*scale.shape, 32)).reshape(code.shape)


CASES = [  # tokens, heads, d, bits, page, dtype
    (1, 1, 64, 4, 16, "f16"), (1, 2, 256, 4, 16, "f16"), (7, 3, 128, 4, 16, "f32"), (33, 2, 64, 8, 48, "f16"),
    (40, 5, 128, 8, 32, "f16"), (19, 1, 256, 8, 16, "f32"), (70, 2, 256, 4, 64, "f32"), (130, 8, 64, 4, 256, "f16"),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("order", ["run", "scattered"])
def test_write_and_read(amd, case, order):
    import torch
    tokens, heads, d, bits, p, dtype = case
    print("  kv cache", case, order, flush=True)
    k, v = rows(40 + tokens, tokens, heads, d, dtype), rows(50 + tokens, tokens, heads, d, dtype, 0.4)
    count = -(-tokens // p) + 2
    order_of = np.argsort(synth.splitmix64(60, count * p))
    slots = (order_of[:tokens] if order == "scattered" else np.arange(tokens) + 5).astype(np.int64)
    size = amd.kv_page_bytes(heads, d, bits, p)
    before = synth.uniform_u16(61, count * size).astype(np.uint8).reshape(count, size)  # other tokens' bytes stay
    pages = torch.from_numpy(before.copy()).cuda()
    sd = torch.from_numpy(slots).cuda()
    amd.kv_cache_write(pages, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), sd, bits=bits, page_tokens=p)
    assert np.array_equal(pages.cpu().numpy(), expected_pages(before, k, v, slots, bits, p))
    for dt, u in ((torch.float16, ref.U16), (torch.float32, 2.0 ** -24)):
        got = amd.kv_cache_read(pages, sd, heads, d, bits=bits, page_tokens=p, out_dtype=dt)
        for x, g in ((k, got[0]), (v, got[1])):
            code, scale = ref.quantise(x, bits)
            want = ref.rotate(ref.values(code, scale, bits))
            err = np.abs(g.double().cpu().numpy() - want)
            assert np.all(err <= read_bound(code, scale, bits) + u * np.abs(want) + 2.0 ** -25)
            # and near the rows that went in: half a step of the largest scale per rotated element
            step = np.repeat(np.abs(scale.astype(np.float64)), 32, -1).reshape(code.shape)
            assert np.linalg.norm(want - x) <= 1.01 * np.linalg.norm(step) * 0.75


def test_special_groups(amd):
    """zeros, tiny and huge groups, ties of the extreme, non-finite elements"""
    import torch
    d, bits, p = 64, 4, 16
    x = np.zeros((10, 1, d), np.float32)
    x[1, 0, 3] = 1.0                     # one element: every rotated element has the same magnitude
    x[2, 0, :32], x[2, 0, 32:] = -2.0, 3.0
    x[3] = 1e-6
    x[4, 0, 0] = 2.0 ** -24
    x[5, 0, :] = 60000.0
    x[6, 0, 4] = 3e6                     # its scale is beyond fp16
    x[7, 0, 40] = np.nan
    x[8, 0, 2] = np.inf
    x[9, 0, 33] = -np.inf
    for bits in (4, 8):
        pages = torch.zeros((1, amd.kv_page_bytes(1, d, bits, p)), dtype=torch.uint8, device="cuda")
        sd = torch.arange(10, device="cuda")
        xd = torch.from_numpy(x).cuda()
        amd.kv_cache_write(pages, xd, xd, sd, bits=bits, page_tokens=p)
        code, scale = ref.quantise(x, bits)
        kc, vc, ks, vs = ref.page_parts(pages.cpu().numpy()[0], bits, 1, d, p)
        for got_code, got_scale in ((kc, ks), (vc, vs)):
            assert np.array_equal(np.isnan(got_scale[0, :10]), np.isnan(scale[:, 0]))
            fine = ~np.isnan(scale[:, 0])
            assert np.array_equal(got_scale[0, :10][fine].view(np.uint16), scale[:, 0][fine].view(np.uint16))
            keep = np.repeat(fine, 32, -1)
            assert np.array_equal(got_code[0, :10][keep], code[:, 0][keep])
        k, _ = amd.kv_cache_read(pages, sd, 1, d, bits=bits, page_tokens=p, out_dtype=torch.float32)
        k = k.cpu().numpy()[:, 0]
        assert np.all(k[0] == 0)
        bad = np.isnan(scale[:, 0])
        assert np.isnan(k.reshape(10, 2, 32)[bad]).all() and np.isfinite(k.reshape(10, 2, 32)[~bad]).all()
        assert bad[6, 0] == (bits == 4 or 3e6 / np.sqrt(32) / 128 > 65504) and bad[7, 1] and bad[8, 0] and bad[9, 1]


def test_slots_outside_the_cache(amd):
    import torch
    heads, d, bits, p = 2, 128, 4, 16
    x = torch.randn(4, heads, d, device="cuda").half()
    pages = torch.full((2, amd.kv_page_bytes(heads, d, bits, p)), 7, dtype=torch.uint8, device="cuda")
    before = pages.clone()
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    skip = torch.tensor([-1, -5, -(1 << 40), -1], device="cuda")
    amd.kv_cache_write(pages, x, x, skip, bits=bits, page_tokens=p, bad_slots=bad)
    assert torch.equal(pages, before) and bad.item() == 0
    amd.kv_cache_write(pages, x, x, torch.tensor([32, 1 << 40, -1, 33], device="cuda"), bits=bits, page_tokens=p,
                       bad_slots=bad)
    assert torch.equal(pages, before) and bad.item() == 1
    bad.zero_()
    slots = torch.tensor([3, 31, 32, -1], device="cuda")
    k, v = amd.kv_cache_read(pages, slots, heads, d, bits=bits, page_tokens=p, bad_slots=bad)
    assert bad.item() == 1 and torch.isnan(k[2:]).all() and torch.isnan(v[2:]).all()
    assert not torch.isnan(k[:2].float()).any()
    amd.kv_cache_write(pages, x[:0], x[:0], slots[:0], bits=bits, page_tokens=p)


def test_views_and_far_pages(amd):
    """strided rows in and out, and pages beyond 4 GiB"""
    import torch
    heads, d, bits, p = 1, 64, 8, 65536
    size = amd.kv_page_bytes(heads, d, bits, p)
    count = (1 << 32) // size + 3
    pages = torch.zeros((count, size), dtype=torch.uint8, device="cuda")
    tokens = 9
    buf = torch.randn(tokens, 2 * heads * d + 5, device="cuda").half()
    k = buf[:, 1:1 + d].unflatten(1, (1, d))
    v = buf[:, 1 + d:1 + 2 * d].unflatten(1, (1, d))
    slots = torch.tensor([(count - 1) * p + 65535 - 7 * i for i in range(tokens)], device="cuda")
    amd.kv_cache_write(pages, k, v, slots, bits=bits, page_tokens=p)
    out = torch.full((2, heads, tokens, d), float("nan"), device="cuda")
    amd.kv_cache_read(pages, slots, heads, d, bits=bits, page_tokens=p, k=out[0].transpose(0, 1),
                      v=out[1].transpose(0, 1))
    small = torch.zeros((1, amd.kv_page_bytes(heads, d, bits, 16)), dtype=torch.uint8, device="cuda")
    at = torch.arange(tokens, device="cuda")
    amd.kv_cache_write(small, k.contiguous(), v.contiguous(), at, bits=bits, page_tokens=16)
    k2, v2 = amd.kv_cache_read(small, at, heads, d, bits=bits, page_tokens=16, out_dtype=torch.float32)
    assert torch.equal(out[0].transpose(0, 1), k2) and torch.equal(out[1].transpose(0, 1), v2)
