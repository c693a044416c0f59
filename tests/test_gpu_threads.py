"""Host threads that call on one stream with its internal workspace: calls of several launches (a prompt in parts, a long
cached sequence joined apart, a split GEMM) give each thread the bits that it gets alone."""
import ctypes
import threading

import pytest

import synth

pytestmark = pytest.mark.gpu
F16, F32 = 1, 0


def test_calls_of_several_launches_on_one_stream(amd):
    import torch
    L = amd.lib()
    stream = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(9)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731

    def view(t):
        return amd.HeadView(t.data_ptr(), t.shape[1], t.stride(0), t.stride(1))

    def prompt(nk, d, hq, hk):  # in parts
        q, k, v, out = draw(17, hq, d), draw(nk, hk, d), draw(nk, hk, d), draw(17, hq, d)
        assert amd.attention_prompt_workspace_bytes(hq, d, 1, 17, nk) > 0
        starts = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (17, nk)]
        views = [view(t) for t in (q, k, v, out)]

        def call():
            return L.exl3_hip_attention_prompt(*(ctypes.byref(x) for x in views), d, starts[0].data_ptr(),
                                               starts[1].data_ptr(), 1, 17, nk, d ** -0.5, 1, None, 0, stream.cuda_stream)
        return call, out, (q, k, v, starts)

    def cached(n, d, hq, hk):  # joined apart
        p = 64
        count = -(-n // p)
        pages = amd.new_kv_cache(count, hk, d, 4, p)
        amd.kv_cache_write(pages, draw(n, hk, d), draw(n, hk, d), torch.arange(n, device="cuda"), bits=4, page_tokens=p)
        table = torch.arange(count, dtype=torch.int32, device="cuda")[None].contiguous()
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        q, out = draw(1, hq, d), draw(1, hq, d)
        qv, ov = view(q), view(out)

        def call():
            return L.exl3_hip_attention_cached(ctypes.byref(qv), ctypes.byref(ov), d, pages.data_ptr(), count, 4, p, hk,
                                               table.data_ptr(), count, lens.data_ptr(), 1, 1, d ** -0.5, None, 0,
                                               stream.cuda_stream)
        return call, out, (q, pages, table, lens)

    def product(k, n, rows):  # split over k
        rec = torch.from_numpy(synth.pack_records(synth.packed_tiles(7, k, n, 4), *synth.layer_scales(7, k, n), 4).view("u1"))
        rec, x, out = rec.cuda(), draw(rows, k), torch.zeros(rows, n, device="cuda")

        def call():
            return L.exl3_hip_mul_mat(rec.data_ptr(), 4, amd.CB_MUL1, k, n, x.data_ptr(), F16, rows, k, out.data_ptr(), F32,
                                      n, None, 0, stream.cuda_stream)
        return call, out, (rec, x)

    jobs = [prompt(3000, 64, 2, 1), prompt(4000, 128, 4, 2), cached(9000, 256, 4, 1), cached(14000, 128, 10, 2),
            product(2048, 512, 64)]
    torch.cuda.synchronize()
    want = []
    for call, out, _ in jobs:  # alone, and twice so that the workspace has its size
        for _ in range(2):
            assert call() == 0
        torch.cuda.synchronize()
        want.append(out.clone())
    failed = []

    def work(i):
        for _ in range(60):
            if jobs[i][0]() != 0:
                failed.append(i)

    for turn in range(5):
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not failed
        for i, (_, out, _) in enumerate(jobs):
            assert torch.equal(out, want[i]), (turn, i)
