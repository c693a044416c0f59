"""exl3_hip_delta_rule against its recurrence in 64 bits where rows, gates and epsilons differ widely within 64 rows."""
import numpy as np
import pytest

import linear_attention_ref as ref
from test_gpu_delta_rule import cuda, draw, inputs, starts_of

pytestmark = pytest.mark.gpu


def compare(amd, d, lens, states, eps, packed=True, chunk=64, scale=None, **kw):
    """out and states of a call that goes on from every state, in place, against the recurrence's; `chunk` None: a call
    that goes row by row"""
    f = {k: None if x is None else x.astype(np.float64) for k, x in d.items()}
    scale = d["q"].shape[2] ** -0.5 if scale is None else scale
    slots = np.arange(len(lens), dtype=np.int32)[::-1].copy()
    want, after, bound, off = ref.delta_rule(f["q"], f["k"], f["v"], f["g"], f["beta"], lens, float(np.float32(scale)),
                                             states.astype(np.float64), slots, slots, f["a_log"], f["dt_bias"],
                                             None if eps is None else float(np.float32(eps)), chunk=chunk)
    t, pool = {k: cuda(x) for k, x in d.items()}, cuda(states)
    where = dict(starts=starts_of(lens)) if packed else dict(sequences=len(lens))
    got = amd.delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], t["a_log"], t["dt_bias"], states=pool,
                         slots_in=cuda(slots), slots_out=cuda(slots), scale=scale, qk_eps=eps, **where, **kw)
    for name, x, w, top in (("out", got.cpu().numpy().astype(np.float64), want,
                             bound + ref.rounded(np.abs(want) + bound, "float16")),
                            ("states", pool.cpu().numpy().astype(np.float64), after, off + ref.E32 * np.abs(after))):
        assert np.all(np.isfinite(x)), name
        err = np.abs(x - w)
        print(f"  {name}: largest error {err.max(initial=0):.2e} of {np.abs(w).max(initial=0):.2e}, "
              f"{np.max(err / top, initial=0):.2f} of its bound")
        assert np.all(err <= top), name


# A key of length |k| has 1 / |k| among the factors of its row: they spread as the lengths do.
@pytest.mark.parametrize("eps", [1e-6, 1e-12, 1e-16, 1e-24, 1e-36])
@pytest.mark.parametrize("n", [14, 64, 150])
@pytest.mark.parametrize("dk,dv", [(128, 16), (64, 48)])
def test_rows_of_zeros(amd, dk, dv, n, eps):
    """keys and queries of nothing, as padding rows give: they leave the state as it is"""
    d = inputs(31, n, 2, 2, dk, dv)
    d["k"][[3, 5, n - 1]] = 0
    d["q"][[4, 5]] = 0
    compare(amd, d, [n], draw(32, (1, 2, dk, dv), 0.5), eps, chunk=64 if n >= 16 else None)


@pytest.mark.parametrize("eps", [1e-6, 1e-12, 0.0])
@pytest.mark.parametrize("least,most", [(-12, 10), (-20, 12)])
@pytest.mark.parametrize("n", [14, 64, 150])
@pytest.mark.parametrize("dk,dv", [(128, 16), (64, 48)])
def test_rows_of_many_lengths(amd, dk, dv, n, least, most, eps):
    d = inputs(33, n, 2, 2, dk, dv)
    rng = np.random.default_rng(5)
    for name in ("q", "k"):
        by = 2.0 ** rng.integers(least, most + 1, (n, 2, 1))
        x = (d[name].astype(np.float64) * by).astype(np.float16)
        x[..., 0] = np.where(np.any(x, -1), x[..., 0], np.float16(2.0 ** -24))  # no row is empty
        d[name] = x
    compare(amd, d, [n], draw(34, (1, 2, dk, dv), 0.5), eps, chunk=64 if n >= 16 else None)


@pytest.mark.parametrize("eps", [1e-38, 1e-40, 2e-45])
@pytest.mark.parametrize("n", [14, 150])
def test_epsilons_at_the_end_of_their_type(amd, n, eps):
    """1 / sqrt(eps) is finite and its square is not"""
    d = inputs(35, n, 2, 2, 64, 32)
    d["k"][[3, 5, 6, n - 1]] = 0
    d["q"][[4, 5, 7]] = 0
    compare(amd, d, [n], draw(36, (1, 2, 64, 32), 0.5), eps, chunk=64 if n >= 16 else None)


@pytest.mark.parametrize("size", [1.0, 300.0, 3e4, 3e6, 3e8])
@pytest.mark.parametrize("n", [14, 64, 100])
def test_states_emptied_on_the_way(amd, n, size):
    """a gate of -inf: 14 rows go row by row and keep binary32's bits, 64 together the steps of the state ahead of them"""
    d = inputs(37, n, 2, 2, 128, 32, raw=False)
    d["g"][n // 2] = -np.inf
    d["v"][:n // 2] = 0
    compare(amd, d, [n], draw(38, (1, 2, 128, 32)) * np.float32(size), 1e-6, chunk=64 if n >= 16 else None, scale=1e-9)


@pytest.mark.parametrize("n", [14, 64, 150])
@pytest.mark.parametrize("least,most", [(-6, 6), (-13, 13)])
@pytest.mark.parametrize("dk,dv", [(128, 32), (64, 48)])
def test_queries_of_many_lengths_as_they_are(amd, dk, dv, n, least, most):
    """without the norm: rows of P differ as the queries do"""
    d = inputs(39, n, 2, 2, dk, dv, norm=False)
    by = 2.0 ** np.random.default_rng(6).integers(least, most + 1, (n, 2, 1))
    d["q"] = (d["q"].astype(np.float64) * by).astype(np.float16)
    compare(amd, d, [n], draw(40, (1, 2, dk, dv), 0.5), None, chunk=64 if n >= 16 else None, scale=1.0)


@pytest.mark.parametrize("n", [14, 64, 150])
@pytest.mark.parametrize("least,most", [(-3, 3), (-8, 6)])
@pytest.mark.parametrize("dk,dv", [(128, 32), (64, 48)])
def test_keys_of_many_lengths_as_they_are(amd, dk, dv, n, least, most):
    """without the norm: beta |k|^2 is at most 1, as where the recurrence is a contraction"""
    d = inputs(41, n, 2, 2, dk, dv, raw=False, norm=False)
    by = 2.0 ** np.random.default_rng(7).integers(least, most + 1, (n, 2))
    d["k"] = (d["k"].astype(np.float64) * by[..., None]).astype(np.float16)
    d["beta"] = (d["beta"] / np.maximum(1, by * by)).astype(np.float32)
    compare(amd, d, [n], draw(42, (1, 2, dk, dv), 0.5), None, chunk=64 if n >= 16 else None)
