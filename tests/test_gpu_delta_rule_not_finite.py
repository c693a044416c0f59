"""What exl3_hip_delta_rule makes of elements that are not finite: which results they reach and which stay as they are."""
import numpy as np
import pytest

import linear_attention_ref as ref
from test_gpu_delta_rule import cuda, draw, inputs, starts_of

pytestmark = pytest.mark.gpu
LENS = {"rows": [5, 7, 6], "chunks": [70, 150, 80]}
NORM = float(np.float32(1e-6))


def run(amd, d, lens, states):
    t, pool = {k: cuda(x) for k, x in d.items()}, cuda(states)
    slots = cuda(np.arange(len(lens), dtype=np.int32))
    out = amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], starts=starts_of(lens),
                         states=pool, slots_in=slots, slots_out=slots, qk_eps=1e-6)
    return out.cpu().numpy().astype(np.float64), pool.cpu().numpy().astype(np.float64)


def restated(d, lens, states, chunk):
    """the recurrence of finite elements, and bounds that count a |v| of 65,504 in each chunk"""
    f = {k: None if x is None else x.astype(np.float64) for k, x in d.items()}
    slots = np.arange(len(lens), dtype=np.int32)
    want, after, bound, off = ref.delta_rule(f["q"], f["k"], f["v"], f["g"], f["beta"], lens,
                                             float(np.float32(d["q"].shape[2] ** -0.5)), states.astype(np.float64), slots,
                                             slots, f["a_log"], f["dt_bias"], NORM, chunk=chunk)
    if chunk:
        # ||T|| is at most 64: u = T r of |r| <= 1 is u = r - beta S^T k, S <- (1 - beta k k^T) S + k r, where |k| <= 1 and
        # 0 <= beta <= 1, so that S grows by at most 1 a row
        floor = 128 * 2.0 ** -38 * 64 * 65504 * (1 + np.arange(sum(lens)) // 64)[:, None, None]
        bound = bound + d["q"].shape[2] ** -0.5 * floor
        off = off + floor.max()
    return want, after, bound + ref.rounded(np.abs(want) + bound, "float16"), np.broadcast_to(off, after.shape) + ref.E32 * np.abs(after)


@pytest.mark.parametrize("way", list(LENS))
@pytest.mark.parametrize("dv", [16, 64])
@pytest.mark.parametrize("name,what", [(n, x) for n in ("q", "k", "v", "state") for x in (np.inf, -np.inf, np.nan)] +
                         [("g", np.nan), ("beta", np.nan)])  # infinite gates are a gate's ends
def test_what_it_reaches(amd, way, dv, name, what):
    """of the middle sequence and head 0 of two: v and a state their column, q its rows, k, g and beta the head"""
    lens, chunk = LENS[way], 64 if way == "chunks" else None
    n0, n1 = lens[0], lens[0] + lens[1]
    d, states = inputs(41, sum(lens), 2, 2, 64, dv), draw(42, (3, 2, 64, dv), 0.5)
    d["k"] = (np.abs(d["k"]) + np.float16(0.05)).astype(np.float16)  # no key leaves a state's element out
    want, after, top, off = restated(d, lens, states, chunk)
    for row in ((0, 3, 6) if way == "rows" else (0, 20, 40, 63, 64, 100, 149)):
        bad, pool = {k: None if x is None else x.copy() for k, x in d.items()}, states.copy()
        first = n0 + row // 64 * 64  # of the rows taken together
        if name == "state":
            if row:
                continue
            pool[1, 0, 11, 5] = what
        else:
            bad[name][(n0 + row, 0, 5)[:bad[name].ndim]] = what
        got, now = run(amd, bad, lens, pool)
        near = np.zeros(want.shape, bool)  # results that may be other ones
        near[first:n1, 0, 5 if name in ("v", "state") else slice(None)] = True
        if name == "q":
            near[min(first + 64, n1):n1] = False
        assert np.all(np.abs(got - want)[~near] <= top[~near]), (row, "out")
        own = got[n0 + row:n1, 0, 5] if name in ("v", "state") else got[n0 + row, 0] if name == "q" else got[n0 + row:n1, 0]
        assert not np.any(np.isfinite(own)), (row, "its own rows")
        far = np.zeros(after.shape, bool)
        if name != "q":
            far[1, 0, :, 5 if name in ("v", "state") else slice(None)] = True
        assert np.all(np.abs(now - after)[~far] <= off[~far]), (row, "states")
        assert not np.any(np.isfinite(now[far])) or name == "state" and way == "rows", (row, "its own state")
