"""The attention block's Python calls on a stream that is not the current one: outputs come from the memory pool of the
stream that writes them.  Out of the current stream's pool they could be memory that work queued there still reads, and
once freed go to the next allocation there while the call's kernel still writes."""
import pytest

pytestmark = pytest.mark.gpu
D, HQ, HK, P = 128, 4, 2, 16


def calls(amd, torch):
    n = 96
    g = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731
    q, k, v = draw(n, HQ, D), draw(n, HK, D), draw(n, HK, D)
    pages = amd.new_kv_cache(8, HK, D, 4, P)
    slots = torch.arange(n, device="cuda")
    amd.kv_cache_write(pages, k, v, slots, bits=4, page_tokens=P)
    table = torch.arange(6, dtype=torch.int32, device="cuda")[None].contiguous()
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([n], [0, n]))
    w = torch.ones(D, device="cuda")
    cache = dict(bits=4, page_tokens=P)
    return {
        "qk_norm_rope": lambda **s: amd.qk_norm_rope(q, k, q_weight=w, k_weight=w, **s),
        "kv_cache_read": lambda **s: amd.kv_cache_read(pages, slots, HK, D, **cache, **s),
        "attention_cached": lambda **s: (amd.attention_cached(q[-1:], pages, table, lens, HK, **cache, **s),),
        "attention_prompt": lambda **s: (amd.attention_prompt(q, k, v, starts, **s),),
    }


@pytest.mark.parametrize("name", ["qk_norm_rope", "kv_cache_read", "attention_cached", "attention_prompt"])
def test_outputs_are_of_the_given_stream(amd, name):
    import torch
    call = calls(amd, torch)[name]
    want = call()
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    side.wait_stream(current)
    got = call(stream=side)
    assert torch.cuda.current_stream() == current
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    shapes, places = [t.shape for t in got], {t.data_ptr() for t in got}
    del got
    again = [torch.empty(s, dtype=torch.float16, device="cuda") for s in shapes]
    assert not places & {t.data_ptr() for t in again}
    with torch.cuda.stream(torch.cuda.default_stream()):  # and the default stream by its number, which is 0
        zero = call(stream=torch.cuda.default_stream())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(zero, want))


def test_tensors_of_the_host_and_of_two_devices_are_refused(amd):
    import torch
    x = torch.randn(3, 2, 64, device="cuda").half()
    starts = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(AssertionError, match="HIP device"):
        amd.attention_prompt(x, x, x, starts.cpu())
    with pytest.raises(AssertionError, match="HIP device"):
        amd.qk_norm_rope(x.cpu(), None)
    if torch.cuda.device_count() > 1:
        with pytest.raises(AssertionError, match="different devices"):
            amd.attention_prompt(x, x, x, starts.to("cuda:1"))


def test_bits_are_not_cut_to_32_bits(amd):
    import torch
    x = torch.zeros(1, HK, D, dtype=torch.float16, device="cuda")
    pages, slots = amd.new_kv_cache(1, HK, D, 4, P), torch.zeros(1, dtype=torch.int64, device="cuda")
    for bits in (0, 5, (1 << 32) + 4):
        with pytest.raises((AssertionError, amd.Exl3Error)):
            amd.kv_cache_write(pages, x, x, slots, bits=bits, page_tokens=P)
