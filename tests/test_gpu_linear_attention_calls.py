"""How the linear-attention block's calls run: on streams of their own, captured in graphs, with workspaces of the
caller's, two at a time, and over offsets beyond 32 bits."""
import numpy as np
import pytest

import linear_attention_ref as ref

pytestmark = pytest.mark.gpu
NAMES = ["rms_norm", "rms_norm_residual", "short_conv", "delta_step", "delta_chunks"]


def calls(amd, torch, seed=1):
    """each call by its name: (function of stream=, its inputs that a test may change, the states that it changes)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, res, w = draw(97, 4, 128).half(), draw(97, 4, 128), draw(128)
    cx, cw, cs = draw(100, 264).half(), draw(264, 4), draw(7, 3, 264).half()
    q, k, v = draw(200, 2, 128).half(), draw(200, 2, 128).half(), draw(200, 4, 64).half()
    gb, ab, S, L = draw(200, 8), draw(2, 4) - 2, draw(6, 4, 128, 64), draw(6, 4, 128, 64)
    slots = torch.tensor([5, 2, 0, 4], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 70, 71, 100, 200], dtype=torch.int32, device="cuda")
    delta = lambda n, pool, where, s: amd.delta_rule(  # noqa: E731
        q[:n], k[:n], v[:n], gb[:n, :4], gb[:n, 4:], ab[0], ab[1], states=pool, slots_in=slots, slots_out=slots, qk_eps=1e-6,
        **where, **s)
    return {
        "rms_norm": (lambda **s: (amd.rms_norm(x, w, gate=x, **s),), x, None),
        "rms_norm_residual": (lambda **s: amd.rms_norm(x, w, residual=res, **s), x, None),
        "short_conv": (lambda **s: (amd.short_conv(cx, cw, sequences=4, states=cs, slots_in=slots, slots_out=slots, **s),),
                       cx, cs),
        "delta_step": (lambda **s: (delta(8, S, dict(sequences=4), s),), v, S),
        "delta_chunks": (lambda **s: (delta(200, L, dict(starts=starts), s),), v, L),
    }


def same(got, want):
    import torch
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_outputs_are_of_the_given_stream(amd, name):
    """the pool of the stream that writes them: out of the current stream's they could be memory that work queued there
    still reads"""
    import torch
    call, _, states = calls(amd, torch)[name]
    before = None if states is None else states.clone()
    want = call()
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    after = None if states is None else states.clone()
    if states is not None:
        states.copy_(before)
    side.wait_stream(current)
    got = call(stream=side)
    assert torch.cuda.current_stream() == current
    side.synchronize()
    assert same(got, want) and (states is None or torch.equal(states, after))
    shapes, places = [(t.shape, t.dtype) for t in got], {t.data_ptr() for t in got}
    del got
    again = [torch.empty(s, dtype=d, device="cuda") for s, d in shapes]
    assert not places & {t.data_ptr() for t in again}
    if states is not None:
        states.copy_(before)
    torch.cuda.synchronize()
    zero = call(stream=torch.cuda.default_stream())  # the default stream by its number, which is 0
    torch.cuda.synchronize()
    assert same(zero, want)


@pytest.mark.parametrize("name", NAMES)
def test_captured_and_replayed(amd, name):
    """every replay against the eager call, with eager calls and synchronisations between them"""
    import torch
    (call, x, states), (eager, x2, states2) = (calls(amd, torch)[name] for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()  # kernels are loaded and the stream's workspace is there
    side.synchronize()
    eager()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for i in range(4):
        new = torch.randn(x.shape, device="cuda").half()
        x.copy_(new), x2.copy_(new)
        graph.replay()
        want = eager()
        torch.cuda.synchronize()
        assert same(got, want) and (states is None or torch.equal(states, states2)), i


def test_host_tensors_are_refused(amd):
    import torch
    x = torch.zeros(6, 2, 64, dtype=torch.float16, device="cuda")
    g, w = torch.zeros(6, 2, device="cuda"), torch.zeros(128, 4, device="cuda")
    starts = torch.tensor([0, 6], dtype=torch.int32)
    for bad in (lambda: amd.rms_norm(x.cpu()), lambda: amd.rms_norm(x, torch.ones(64)),
                lambda: amd.rms_norm(x, residual=x.cpu()), lambda: amd.short_conv(x.view(6, 128), w.cpu()),
                lambda: amd.short_conv(x.view(6, 128), w, starts=starts), lambda: amd.delta_rule(x, x, x, g, g.cpu()),
                lambda: amd.delta_rule(x, x, x, g, g, starts=starts),
                lambda: amd.delta_rule(x, x, x, g, g, states=torch.zeros(1, 2, 64, 64),
                                       slots_out=torch.zeros(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(AssertionError, match="HIP device"):
            bad()


def delta_args(torch, n, hk=2, hv=4, dk=128, dv=64, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return (draw(n, hk, dk).half(), draw(n, hk, dk).half(), draw(n, hv, dv).half(), draw(n, hv), draw(n, hv), draw(hv),
            draw(hv) - 2)


def test_workspaces_of_the_caller(amd):
    """whatever is in them; the same one for calls of other sizes; a smaller or displaced one is refused"""
    import torch
    sizes = [(200, 1), (90, 3), (640, 2), (17, 1)]
    need = max(amd.delta_rule_workspace_bytes(4, 128, 64, s, n) for n, s in sizes)
    assert need > 0 and amd.delta_rule_workspace_bytes(4, 128, 64, 8, 8) == 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for fill in (0, 255, 0x7C):
        for n, s in sizes:
            args = delta_args(torch, n)
            starts = torch.tensor([0] + [n] * s, dtype=torch.int32, device="cuda")
            want = amd.delta_rule(*args, starts=starts, qk_eps=1e-6)
            assert bool(torch.isfinite(want).all())
            ws.fill_(fill)
            assert torch.equal(amd.delta_rule(*args, starts=starts, qk_eps=1e-6, workspace=ws), want), (fill, n)
            assert torch.equal(amd.delta_rule(*args, starts=starts, qk_eps=1e-6, workspace=ws), want), (fill, n)
    args = delta_args(torch, 200)
    need = amd.delta_rule_workspace_bytes(4, 128, 64, 1, 200)
    for bad in (ws[:need - 1], ws[16:16 + need]):
        with pytest.raises((AssertionError, amd.Exl3Error)):
            amd.delta_rule(*args, workspace=bad)
    for n in (4, 200):  # a call that needs none takes any; rows behind the workspace's last byte stay as they are
        args = delta_args(torch, n)
        need = amd.delta_rule_workspace_bytes(4, 128, 64, 1, n)
        ws.fill_(7)
        amd.delta_rule(*args, workspace=ws[:max(need, 256)])
        assert bool((ws[max(need, 256):] == 7).all())


@pytest.mark.parametrize("own", [False, True])
def test_two_calls_at_once(amd, own):
    """on two streams, each with a workspace of its own or the library's for its stream"""
    import torch
    a, b = (delta_args(torch, n, seed=n) for n in (3000, 2500))
    want = [amd.delta_rule(*t, qk_eps=1e-6) for t in (a, b)]
    ws = [torch.empty(amd.delta_rule_workspace_bytes(4, 128, 64, 1, n), dtype=torch.uint8, device="cuda") if own else None
          for n in (3000, 2500)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [amd.delta_rule(*t, qk_eps=1e-6, workspace=w, stream=s) for t, w, s in zip((a, b), ws, streams)]
        torch.cuda.synchronize()
        assert same(got, want)


def test_states_beyond_32_bits_of_elements(amd):
    """slots at both ends of a pool of 2^31 elements and more"""
    import torch
    slots = 8200  # of 2^18 elements
    pool = torch.empty(slots, 16, 128, 128, dtype=torch.float32, device="cuda")
    small = torch.zeros(3, 16, 128, 128, device="cuda")
    far = torch.tensor([slots - 1, 0, slots - 2], dtype=torch.int32, device="cuda")
    near = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    for n in (3, 150):
        args = delta_args(torch, n, 16, 16, 128, 128)
        small.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
        for f, m in zip((slots - 1, 0, slots - 2), (2, 0, 1)):
            pool[f].copy_(small[m])
        got = amd.delta_rule(*args, sequences=3, states=pool, slots_in=far, slots_out=far, qk_eps=1e-6)
        want = amd.delta_rule(*args, sequences=3, states=small, slots_in=near, slots_out=near, qk_eps=1e-6)
        assert torch.equal(got, want)
        assert all(torch.equal(pool[f], small[m]) for f, m in zip((slots - 1, 0, slots - 2), (2, 0, 1)))


def spread(torch, t, stride):
    """t's rows at a stride of elements, in memory of their own"""
    rows, width = t.shape[0], t[0].numel()
    base = torch.empty((rows - 1) * stride + width, dtype=t.dtype, device="cuda")
    v = base.as_strided((rows,) + t.shape[1:], (stride,) + t.stride()[1:])
    v.copy_(t)
    return v


@pytest.mark.parametrize("stride", [1 << 24, (1 << 24) + 8], ids=["2^24", "2^24+8"])
def test_rows_beyond_32_bits_of_elements(amd, stride):
    """150 rows that lie 2^24 elements apart: beyond that the chunks hand over to the row-by-row kernel"""
    import torch
    q, k, v, *gates = delta_args(torch, 150, 1, 1, 64, 16)
    want = amd.delta_rule(q, k, v, *gates, qk_eps=1e-6)
    out = spread(torch, torch.zeros_like(v), stride)
    for far in ((spread(torch, q, stride), k, v), (q, spread(torch, k, stride), v), (q, k, spread(torch, v, stride))):
        got = amd.delta_rule(*far, *gates, qk_eps=1e-6, out=out)
        row_by_row = stride > 1 << 24
        f = lambda t: t.cpu().numpy().astype(np.float64)  # noqa: E731
        if not row_by_row:
            assert torch.equal(got, want)
        ex, _, bound, _ = ref.delta_rule(f(q), f(k), f(v), f(gates[0]), f(gates[1]), [150], 0.125, None, None, None,
                                         f(gates[2]), f(gates[3]), float(np.float32(1e-6)), chunk=64)
        assert np.all(np.abs(f(got) - ex) <= bound + ref.rounded(np.abs(ex) + bound, "float16"))
        del far
    x = torch.randn(150, 64, device="cuda").half()
    w, far = torch.randn(64, 4, device="cuda"), spread(torch, x, stride)
    wide = spread(torch, torch.zeros_like(x), stride)
    amd.short_conv(far, w, out=wide)
    assert torch.equal(wide, amd.short_conv(x, w))
    amd.rms_norm(far, residual=far, out=wide)
    assert torch.equal(wide, amd.rms_norm(x, residual=x)[0])
