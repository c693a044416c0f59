"""Tensors that the linear-attention block's binding takes: strides that a call does not use, and places of 16 bytes."""
import pytest

pytestmark = pytest.mark.gpu


def test_one_row_of_gates_has_any_stride(amd):
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = draw(1, 2, 64).half(), draw(1, 2, 64).half(), draw(1, 4, 32).half()
    wide, beta = draw(1, 11), draw(1, 4)
    want = amd.delta_rule(q, k, v, wide[:, 2:6].contiguous(), beta)
    for a, b in ((wide[:, 2:6], beta), (wide[:, 2:6].contiguous(), wide.new_zeros(1, 9)[:, :4].copy_(beta))):
        assert torch.equal(amd.delta_rule(q, k, v, a, b), want)
    none = [t[:0] for t in (q, k, v, wide[:, 2:6], beta)]
    assert amd.delta_rule(*none).shape == (0, 4, 32)
    two = [t.repeat(2, *[1] * (t.dim() - 1)) for t in (q, k, v, wide, beta)]
    with pytest.raises(AssertionError, match="row stride"):
        amd.delta_rule(*two[:3], two[3][:, 2:6], two[4])


@pytest.mark.parametrize("off", [4, 8, 12, 1])
def test_fp32_rows_at_places_of_16_bytes(amd, off):
    """eight channels at a time lie at 16-byte places that are none of 32"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(off + 37 * 80, generator=g, device="cuda")
    x, w = base[off:].view(37, 80)[:, :40], torch.randn(40, 4, generator=g, device="cuda")
    dense = x.contiguous()
    out = torch.zeros(off + 37 * 48, device="cuda")[off:].view(37, 48)
    amd.short_conv(x, w, bias=w[:, 0].contiguous(), sequences=1, out=out[:, :40])
    assert torch.equal(out[:, :40], amd.short_conv(dense, w, bias=w[:, 0].contiguous()))
    assert bool((out[:, 40:] == 0).all())
