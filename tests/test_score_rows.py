"""More of the log probabilities and their gradient: calls whose outputs are not
all wanted."""
import numpy as np
import pytest

import test_score as S
import train_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


@pytest.mark.parametrize("n,V,top", [(1, 8185, 5), (1, 151936, 1), (3, 40001, 20), (700, 9000, 64)])
def test_alternatives_that_nobody_takes(gpu, n, V, top):
    """n_top with neither array of alternatives, in the workspace queried for n_top"""
    import hiprt
    rng, bits, l = S.make(n, V, "bf16", 11)
    tokens = rng.integers(0, V, (n, 1))
    ref = R.score(l, S.temperatures(0.7, n), None, tokens, 0)
    with R.Arena() as D:
        lg, tok, lp, st = D.put(bits), D.put(tokens.astype(np.int32)), D.room(4 * n, 0xee), D.room(8 * n, 0xee)
        W = gpu.Workspace(gpu.lib().d3s_logprob_workspace_bytes(gpu.DTYPE_BF16, n, V, top))
        D.held.append(W.buf)
        assert gpu.logprob_raw(lg.ptr, gpu.DTYPE_BF16, n, V, V, 0.7, None, tok.ptr, 1, lp.ptr, None, st.ptr, top,
                               workspace=W.arg()) == 0
        hiprt.synchronize()
        R.assert_near(lp.download((n, 1), np.float32), ref["logprobs"], R.score_tol(ref, ref["logprobs"]))
        R.assert_near(st.download((n, 2), np.float32)[:, 0], ref["m"], 0)


@pytest.mark.parametrize("per_row", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [3, 4097, 60001])
def test_temperatures_that_are_not_finite(gpu, V, dtype, per_row):
    """infinities of both signs and NaN refuse a row, and its gradient"""
    n, inf = 6, np.inf
    T = np.float32([-inf, 0.8, inf, -inf, np.nan, -1e30])
    rng, bits, l = S.make(n, V, dtype, 12)
    l[3, 1] = -inf
    bits, l = R.to_bits(l, dtype)
    tokens = np.stack([rng.integers(0, V, n), np.full(n, -1)], 1)
    # (the plain form clamps before it looks: any temperature that it refuses stands for those)
    ref = R.score(l, np.where(np.isfinite(T), T, inf).astype(np.float64), None, tokens, 3)
    refused = ~np.isfinite(T)
    assert np.array_equal(ref["refused"], refused)
    g, gH = rng.standard_normal((n, 2)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    dx, err = R.score_grad(ref, tokens, g.astype(np.float64), gH)
    dx[refused] = np.where(np.isneginf(l[refused]), 0.0, np.nan)
    if per_row:
        S.check(S.run(gpu, bits, T, None, tokens, 3), ref)
        S.check_grad(S.run_grad(gpu, bits, T, None, tokens, ref, g, gH), dx, np.nan_to_num(err, nan=0.0) + 1e-37)
        return
    for r in range(n):
        one = {k: v[r:r + 1] for k, v in ref.items()}
        S.check(S.run(gpu, bits[r:r + 1], T[r], None, tokens[r:r + 1], 3), one)


def flat_rows(n, V, order):
    """rows whose logits share their upper 16 bits, each value a few times"""
    row = np.float32(1) + (np.arange(V) // (V // 65536 + 1)).astype(np.float32) * np.float32(2.0 ** -23)
    row = row[::-1] if order == "falling" else np.random.default_rng(13).permutation(row) if order == "mixed" else row
    return np.ascontiguousarray(np.broadcast_to(row, (n, V)))


@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("n,V", [(2, 60000), (700, 30011), (1100, 9001)])
def test_alternatives_of_rows_that_rise_a_little(gpu, n, V, order, top):
    l = flat_rows(n, V, order)
    tokens = np.zeros((n, 1), np.int64)
    S.check(S.run(gpu, l, 1.0, None, tokens, top), R.score(l.astype(np.float64), np.ones(n), None, tokens, top))


@pytest.mark.parametrize("top", [1, 20, 64])
def test_passes_over_rows_that_rise_a_little(gpu, top):
    """the segment's passes for its alternatives are few whatever its order: rising rows
    take the time of falling ones, whose first pass files the best, a few times over
    (each pass that files the first of those that reach leaves out 448 elements of
    131072 at most, 292 passes)"""
    import time

    import hiprt
    n, V = 600, 131072
    times = {}
    with R.Arena() as D:
        tok, lp, ids = D.put(np.zeros((n, 1), np.int32)), D.room(4 * n), D.room(4 * n * top)
        for order in ("falling", "rising"):
            lg = D.put(flat_rows(n, V, order))
            for _ in range(4):
                hiprt.synchronize()
                start = time.perf_counter()
                assert gpu.logprob_raw(lg.ptr, gpu.DTYPE_F32, n, V, V, 1.0, None, tok.ptr, 1, lp.ptr, None, None, top,
                                       ids.ptr) == 0
                hiprt.synchronize()
                times[order] = min(times.get(order, 1e9), time.perf_counter() - start)
    assert times["rising"] < 12 * times["falling"], times


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_more_rows_than_a_launch(gpu, dtype):
    """2^22 workgroups a launch, one a row: the second launch's rows, tokens,
    temperatures, statistics, alternatives and gradients"""
    import hiprt
    n, V = (1 << 22) + 5, 3
    rng = np.random.default_rng(16)
    code = gpu.DTYPE_F32 if dtype == "f32" else gpu.DTYPE_BF16
    bits, l = R.to_bits(rng.standard_normal((n, V)).astype(np.float32), dtype)
    T = rng.uniform(0.5, 1.5, n).astype(np.float32)
    tokens, banned = rng.integers(0, V, (n, 1)), rng.integers(-1, V, n)
    g, gH = rng.standard_normal((n, 1)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    with R.Arena() as D:
        lg, tok, temp, ban = D.put(bits), D.put(tokens.astype(np.int32)), D.put(T), D.put(banned.astype(np.int32))
        lp, ent, st = D.room(4 * n, 0xee), D.room(4 * n, 0xee), D.room(8 * n, 0xee)
        ids, tlp, grad = D.room(8 * n, 0xee), D.room(8 * n, 0xee), D.room(bits.nbytes, 0xee)
        assert gpu.logprob_raw(lg.ptr, code, n, V, V, ("ptr", temp.ptr), ban.ptr, tok.ptr, 1, lp.ptr, ent.ptr, st.ptr, 2,
                               ids.ptr, tlp.ptr) == 0
        assert gpu.logprob_backward_raw(lg.ptr, code, n, V, V, ("ptr", temp.ptr), ban.ptr, tok.ptr, 1, st.ptr, ent.ptr,
                                        D.put(g).ptr, D.put(gH).ptr, grad.ptr, V) == 0
        hiprt.synchronize()
        got = dict(logprobs=lp.download((n, 1), np.float32), H=ent.download((n,), np.float32),
                   stats=st.download((n, 2), np.float32), top_ids=ids.download((n, 2), np.int32),
                   top_logprobs=tlp.download((n, 2), np.float32), counters=np.zeros(4, np.uint32))
        dl = grad.download((n, V), bits.dtype)
    # whole, coarsely: no row is another's
    x = np.where(np.arange(V) == banned[:, None], -np.inf, l) / T[:, None]
    x -= x.max(1, keepdims=True)
    logp = x - np.log(np.exp(x).sum(1, keepdims=True))
    R.assert_near(got["logprobs"], np.take_along_axis(logp, tokens, 1), 1e-4)
    # on both sides of the launches' border, and here and there
    at = np.unique(np.concatenate([np.arange(300), np.arange(n - 300, n), rng.integers(0, n, 2000)]))
    ref = R.score(l[at], T[at].astype(np.float64), banned[at], tokens[at], 2)
    S.check({k: v if k == "counters" else v[at] for k, v in got.items()}, ref)
    dx, err = R.score_grad(ref, tokens[at], g[at].astype(np.float64), gH[at])
    # (from the kernel's own fp32 statistics: their roundings move every p alike)
    S.check_grad(dl[at], dx, 2 * err)
