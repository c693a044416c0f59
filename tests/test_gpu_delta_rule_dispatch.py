"""exl3_hip_delta_rule at the borders between its ways, row by row and in chunks, against its recurrence in 64 bits."""
import numpy as np
import pytest

from test_gpu_delta_rule import cuda, draw, inputs, starts_of
from test_gpu_delta_rule_ranges import compare

pytestmark = pytest.mark.gpu


def goes_in_chunks(amd, d, lens, packed):
    """a call that does refuses a workspace of 256 bytes, one that goes row by row uses none"""
    import torch
    t = {k: cuda(x) for k, x in d.items()}
    where = dict(starts=starts_of(lens)) if packed else dict(sequences=len(lens))
    try:
        amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], qk_eps=1e-6,
                       workspace=torch.empty(256, dtype=torch.uint8, device="cuda"), **where)
    except amd.Exl3Error:
        return True
    return False


# heads of q and k, of v, their sizes; sequences, rows of each; whether they are taken 64 at a time
@pytest.mark.parametrize("hk,hv,dk,dv,seqs,n,chunks", [
    (2, 2, 128, 48, 3, 65, True), (1, 3, 64, 96, 2, 130, True), (2, 4, 128, 128, 5, 16, True),
    (2, 4, 128, 128, 5, 15, False), (2, 2, 64, 64, 4, 64, True), (2, 8, 128, 256, 4, 15, False),
    (2, 8, 128, 256, 4, 16, False), (2, 8, 128, 256, 4, 23, False), (2, 8, 128, 256, 4, 24, True),
    (1, 7, 128, 256, 4, 16, True), (4, 16, 64, 256, 4, 70, True), (4, 16, 128, 256, 4, 66, True)])
def test_sequences_of_one_length(amd, hk, hv, dk, dv, seqs, n, chunks):
    d = inputs(51, seqs * n, hk, hv, dk, dv)
    assert goes_in_chunks(amd, d, [n] * seqs, False) == chunks
    compare(amd, d, [n] * seqs, draw(52, (seqs, hv, dk, dv), 0.5), 1e-6, packed=False, chunk=64 if chunks else None)


# packed ones: 16 rows in all and two a sequence, on the average
@pytest.mark.parametrize("lens,chunks", [([15], False), ([16], True), ([1] * 15, False), ([2] * 7, False), ([2] * 8, True),
                                         ([1] * 70 + [68], False), ([1] * 70 + [72], True), ([1] * 101 + [99], False)],
                         ids=["15", "16", "15x1", "7x2", "8x2", "70x1+68", "70x1+72", "101x1+99"])
def test_packed_sequences(amd, lens, chunks):
    """among them prompts of more than 64 rows that go row by row"""
    d = inputs(53, sum(lens), 1, 2, 64, 32)
    assert goes_in_chunks(amd, d, lens, True) == chunks
    compare(amd, d, lens, draw(54, (len(lens), 2, 64, 32), 0.5), 1e-6, chunk=64 if chunks else None)


@pytest.mark.parametrize("seqs,n", [(65536, 1), (65536, 2), (9000, 9)])
def test_as_many_sequences_as_there_may_be(amd, seqs, n):
    """packed ones, whose places every workgroup looks for, and the same without starts, bit for bit; states at their ends"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    starts = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * n
    slots = torch.randperm(seqs, generator=g, device="cuda").to(torch.int32)
    x, w, old = draw(seqs * n, 8).half(), draw(8, 4), draw(seqs, 3, 8).half()
    a, b = old.clone(), old.clone()
    got = amd.short_conv(x, w, starts=starts, states=a, slots_in=slots, slots_out=slots)
    want = amd.short_conv(x, w, sequences=seqs, states=b, slots_in=slots, slots_out=slots)
    assert torch.equal(got, want) and torch.equal(a, b)
    q, k, v = (draw(seqs * n, 1, d).half() for d in (64, 64, 16))
    gates, old = draw(seqs * n, 2), draw(seqs, 1, 64, 16)
    a, b = old.clone(), old.clone()
    decay, beta = -gates[:, :1].abs(), gates[:, 1:].sigmoid()
    got = amd.delta_rule(q, k, v, decay, beta, starts=starts, states=a, slots_in=slots, slots_out=slots, qk_eps=1e-6)
    if n < 8:  # row by row both
        want = amd.delta_rule(q, k, v, decay, beta, sequences=seqs, states=b, slots_in=slots, slots_out=slots, qk_eps=1e-6)
    else:  # in chunks, a thousand sequences a call
        want = torch.cat([amd.delta_rule(*(t[i * n:(i + 1000) * n] for t in (q, k, v, decay, beta)), starts=starts[:1001],
                                         states=b, slots_in=slots[i:i + 1000], slots_out=slots[i:i + 1000], qk_eps=1e-6)
                          for i in range(0, seqs, 1000)])
    assert torch.equal(got, want) and torch.equal(a, b)
