"""Verification of drafted tokens (d3s_verify, d3s_verify_ranked) against a plain form in
64 bits.  Tokens and counts are equal: the uniforms stay 1e-4 off p / q, and the draw's
sums are 64-bit on both sides.  accept = min(1, p / q): p and q are each exp of an
argument that is off by 2 u of itself (below 60 here in size where p is not 0 in fp32 terms that
matter), over a sum off by (adds + 8) u relative."""
import math

import numpy as np
import pytest

import step_ref as SR
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


def run(gpu, target, draft, drafted, lengths, T, Td, u_accept, u_draw, td="bf16", dd="bf16", pad=0, lead=0, stream=None,
        workspace=None):
    """host float arrays in (target [n, L + 1, V], draft [n, L, V] or None); (tokens,
    n_accepted, accept, counters) and the values the library saw"""
    import ctypes
    import hiprt
    n, L1, V = target.shape
    L = L1 - 1
    with R.Arena() as D:
        tb, tv = R.to_bits(target.reshape(-1, V), td)
        stride = V + pad
        es = tb.itemsize
        t = D.put(R.with_stride(tb, stride, lead))
        d, dv = None, None
        if draft is not None:
            db, dv = R.to_bits(draft.reshape(-1, V), dd)
            d = D.put(R.with_stride(db, stride, lead) if L else np.zeros(4, db.dtype))
            dv = dv.reshape(n, L, V)
        i32 = lambda a: D.put(np.asarray(a, np.int32)) if np.size(a) else D.room(4)  # noqa: E731
        f32 = lambda a: D.put(np.asarray(a, np.float32)) if np.size(a) else D.room(4)  # noqa: E731
        temp = lambda v: ("ptr", f32(v).ptr) if np.ndim(v) else float(v)  # noqa: E731
        tokens, acc, accept = D.room(4 * n * L1, 0x77), D.room(4 * n, 0x77), D.room(4 * n * max(L, 1), 0x77)
        counters = D.room(16).zero()
        args = dict(target=t.ptr + lead * es, target_dtype=0 if td == "f32" else 1, target_stride=stride,
                    draft=d.ptr + lead * (4 if dd == "f32" else 2) if d else None, draft_dtype=0 if dd == "f32" else 1,
                    draft_stride=stride, n_seqs=n, n_draft=L, vocab=V, drafted=i32(drafted).ptr,
                    lengths=None if lengths is None else i32(lengths).ptr, temperature=temp(T), draft_temperature=temp(Td),
                    u_accept=f32(u_accept).ptr, u_draw=f32(u_draw).ptr, tokens=tokens.ptr, n_accepted=acc.ptr,
                    accept=accept.ptr, counters=counters.ptr)
        if workspace == "own":
            W = gpu.Workspace(gpu.lib().d3s_verify_workspace_bytes(ctypes.byref(gpu.verify_params(**args))))
            D.held.append(W.buf)
            workspace = W.arg()
        assert gpu.verify_raw(**args, stream=stream, workspace=workspace) == 0
        hiprt.synchronize()
        return (tokens.download((n, L1), np.int32), acc.download((n,), np.int32),
                accept.download((n, L), np.float32) if L else np.zeros((n, 0), np.float32),
                counters.download((4,), np.uint32)), (tv.reshape(n, L1, V), dv)


def check(got, want, V):
    tokens, n_acc, accept, counters = got
    ref_tokens, ref_acc, ref_accept, bad, masked = want
    assert np.array_equal(n_acc, ref_acc), (n_acc, ref_acc)
    assert np.array_equal(tokens, ref_tokens), np.argwhere(tokens != ref_tokens)[:5]
    # p / q: both sums and exponents, 2 (adds + 2 * 60 + 8) steps relative; below 2^-126 p is 0 or subnormal
    R.assert_near(accept, ref_accept, SR.U * 2 * (R.adds(V) + 128) * np.abs(ref_accept) + 1e-30, "accept")
    assert counters[0] == bad and counters[1] == masked


def inputs(n, L, V, seed, spread=2.0, near=0.8):
    rng = np.random.default_rng([n, L, V, seed])
    target = rng.standard_normal((n, L + 1, V)).astype(np.float32) * spread
    draft = (target[:, :L] + near * rng.standard_normal((n, L, V))).astype(np.float32)
    w = SR.probs(draft.astype(np.float64), 1.0).reshape(n * L, V)
    drafted = np.array([rng.choice(V, p=r / r.sum()) for r in w], np.int64).reshape(n, L) if n * L else np.zeros((n, L), int)
    u = lambda *s: (rng.integers(0, 1 << 24, s) * 2.0 ** -24).astype(np.float32)  # noqa: E731
    return target, draft, drafted, u(n, L), u(n), rng


def both(gpu, target, draft, drafted, lengths, T, Td, ua, ud, td="bf16", dd="bf16", **kw):
    n, L1, V = target.shape
    full = lambda v: np.broadcast_to(np.asarray(v, np.float32).astype(np.float64), (n,))  # noqa: E731
    tv = R.to_bits(target.reshape(-1, V), td)[1].reshape(target.shape)
    dv = None if draft is None else R.to_bits(draft.reshape(-1, V), dd)[1].reshape(draft.shape)
    ua = SR.keep_off_borders(tv, dv, drafted, full(T), full(Td), ua)
    got, _ = run(gpu, target, draft, drafted, lengths, T, Td, ua, ud, td, dd, **kw)
    want = SR.verify(tv, dv, drafted, lengths, full(T), full(Td), ua, ud)
    check(got, want, V)
    return got


@pytest.mark.parametrize("n,L,V,td,dd,pad,lead", [
    (1, 4, 4097, "bf16", "bf16", 0, 0), (3, 0, 50, "bf16", "bf16", 0, 0), (5, 1, 1, "f32", "bf16", 3, 1),
    (2, 8, 1000, "f32", "f32", 1, 1), (7, 3, 4097, "bf16", "f32", 7, 3), (2, 64, 37, "f32", "bf16", 0, 0),
    (300, 2, 129, "bf16", "bf16", 0, 1), (3, 2, 8192, "bf16", "bf16", 0, 0), (3, 3, 8193, "f32", "f32", 0, 0),
    (2, 2, 16385, "bf16", "bf16", 5, 2), (4, 2, 40001, "bf16", "f32", 0, 0), (20, 3, 20000, "bf16", "bf16", 8, 0),
    (3, 2, 151936, "bf16", "bf16", 0, 0), (1, 1, 300007, "f32", "f32", 1, 0)])
def test_against_64_bits(gpu, n, L, V, td, dd, pad, lead):
    target, draft, drafted, ua, ud, rng = inputs(n, L, V, 1)
    lengths = rng.integers(0, L + 1, n) if n > 2 else None
    T = (0.5 + rng.random(n)).astype(np.float32) if n % 2 else 1.0
    both(gpu, target, draft, drafted, lengths, T, 0.8, ua, ud, td, dd, pad=pad, lead=lead)


@pytest.mark.parametrize("V", [20, 4097, 30000])
def test_certain_drafts(gpu, V):
    target, draft, _, ua, ud, _ = inputs(40, 3, V, 2, spread=3.0)
    drafted = target[:, :3].argmax(-1)  # likely enough to be accepted now and then
    got = both(gpu, target, None, drafted, None, 0.7, 1.0, ua, ud)
    assert (got[1] > 0).any() and (got[1] < 3).any()


@pytest.mark.parametrize("V", [64, 5000, 20000])
def test_masks_and_refused_rows(gpu, V):
    """masked places, rows masked everywhere, the type's lowest value, NaN and +inf
    before and behind the place where the sequence ends"""
    n, L = 24, 3
    target, draft, drafted, ua, ud, rng = inputs(n, L, V, 3)
    low = np.float32(np.finfo(np.float32).min)
    for b in range(n):
        k = b % 12
        some = rng.random(V) < 0.4
        if k == 0:
            target[b, :, some] = -np.inf
        elif k == 1:
            draft[b, :, some] = -np.inf
        elif k == 2:
            target[b, 1] = -np.inf
        elif k == 3:
            draft[b, 0] = -np.inf
        elif k == 4:
            target[b, :, some] = low
        elif k == 5:
            target[b, 1, V // 2] = np.nan
        elif k == 6:
            target[b, L, 0] = np.inf
        elif k == 7:
            draft[b, 1, V - 1] = np.nan
        elif k == 8:  # everything accepted, then a masked row
            target[b, :L] = draft[b]
            ua[b] = 0.0
            target[b, L] = -np.inf
        elif k == 9:  # nothing accepted: what follows is not looked at
            ua[b, 0] = np.float32(1 - 2.0 ** -24)
            target[b, 0, drafted[b, 0]] = -np.inf
            target[b, 1:] = np.nan
            draft[b, 1:] = np.inf
        elif k == 10:
            drafted[b] = [-1, V, 5 % V]
        else:
            target[b, :, some] = low
            draft[b, :, ~some] = low
    both(gpu, target, draft, drafted, None, 1.0, 1.0, ua, ud, "f32", "f32")
    got = both(gpu, target, draft, drafted, None, 1.0, 1.0, ua, ud)
    assert got[3][0] > 0 and got[3][1] > 0


@pytest.mark.parametrize("V", [100, 4097, 20000])
def test_temperatures(gpu, V):
    n, L = 8, 3
    target, draft, drafted, ua, ud, _ = inputs(n, L, V, 4)
    drafted[:4] = draft[:4].argmax(-1)
    T = np.array([0.0, 1e-6, -3.0, 1e-5, math.nan, math.inf, -math.inf, 100.0], np.float32)
    both(gpu, target, draft, drafted, None, T, T, ua, ud, "f32", "f32")
    both(gpu, target, draft, drafted, None, 1.0, T, ua, ud)


@pytest.mark.parametrize("V", [300, 16384])
def test_the_same_model_accepts_everything(gpu, V):
    target, _, _, ua, ud, rng = inputs(10, 4, V, 5)
    drafted = rng.integers(0, V, (10, 4))
    ua[:] = np.float32(1 - 2.0 ** -24)
    got, _ = run(gpu, target, target[:, :4].copy(), drafted, None, 0.9, 0.9, ua, ud, "f32", "f32")
    assert (got[1] == 4).all() and np.array_equal(got[0][:, :4], drafted) and (got[2] == 1.0).all()


@pytest.mark.parametrize("V", [50, 9000])
def test_the_ends_of_the_draw(gpu, V):
    target, draft, drafted, ua, ud, _ = inputs(6, 2, V, 6)
    ud[:3], ud[3:] = 0.0, np.float32(1 - 2.0 ** -24)
    target[:, :, :3] = -np.inf
    target[:, :, V - 4:] = -np.inf
    both(gpu, target, draft, drafted, None, 1.0, 1.0, ua, ud, "f32", "f32")


@pytest.mark.parametrize("certain", [False, True])
def test_tokens_are_distributed_as_the_targets(gpu, certain):
    """the first token of many sequences on the same logits: each frequency within five
    deviations of sqrt(p (1 - p) / n)"""
    n, V = 40000, 12
    rng = np.random.default_rng(7)
    t, d = rng.standard_normal(V) * 1.5, rng.standard_normal(V) * 1.5
    p, q = SR.probs(R.to_bits(t, "bf16")[1], 1.0), SR.probs(R.to_bits(d, "bf16")[1], 1.0)
    drafted = np.full((n, 1), 3) if certain else rng.choice(V, (n, 1), p=q / q.sum())
    u = lambda *s: (rng.integers(0, 1 << 24, s) * 2.0 ** -24).astype(np.float32)  # noqa: E731
    got, _ = run(gpu, np.broadcast_to(t, (n, 2, V)).astype(np.float32),
                 None if certain else np.broadcast_to(d, (n, 1, V)).astype(np.float32), drafted, None, 1.0, 1.0, u(n, 1), u(n))
    freq = np.bincount(got[0][:, 0], minlength=V) / n
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-3 * p).all(), (freq, p)


# ---- ranked candidates ----
def ranked_rows(rows, k, V, rng, cut=0.9):
    """as d3s_sample writes them: (cand, probs)"""
    cand, probs = np.zeros((rows, k), np.int32), np.zeros((rows, k), np.float32)
    for r in range(rows):
        l = rng.standard_normal(V) * 2  # noqa: E741
        order = np.argsort(-l)[:k]
        p = SR.probs(l, 1.0)[order]
        c = np.cumsum(p)
        kept = np.where((c > cut) & (np.arange(k) > 0), 0.0, p)
        cand[r], probs[r] = order, (kept / kept.sum()).astype(np.float32)
    return cand, probs


def run_ranked(gpu, tc, tp, dc, dp, drafted, lengths, ua, ud, V=None):
    import hiprt
    n, L = drafted.shape
    with R.Arena() as D:
        put = lambda a, t: D.put(np.ascontiguousarray(a, t)) if np.size(a) else D.room(4)  # noqa: E731
        tokens, acc, accept = D.room(4 * n * (L + 1), 0x77), D.room(4 * n, 0x77), D.room(4 * n * max(L, 1), 0x77)
        counters = D.room(16).zero()
        rc = gpu.verify_ranked_raw(put(tc, np.int32).ptr, put(tp, np.float32).ptr, tc.shape[-1],
                                   None if dc is None else put(dc, np.int32).ptr, None if dp is None else put(dp, np.float32).ptr,
                                   0 if dc is None else dc.shape[-1], n, L, put(drafted, np.int32).ptr,
                                   None if lengths is None else put(lengths, np.int32).ptr, put(ua, np.float32).ptr,
                                   put(ud, np.float32).ptr, tokens.ptr, acc.ptr, accept=accept.ptr, counters=counters.ptr)
        assert rc == 0
        hiprt.synchronize()
        return (tokens.download((n, L + 1), np.int32), acc.download((n,), np.int32),
                accept.download((n, L), np.float32) if L else np.zeros((n, 0), np.float32), counters.download((4,), np.uint32))


def ranked_ref(tc, tp, dc, dp, drafted, lengths, ua, ud):
    n, L = drafted.shape
    tc, tp = tc.reshape(n, L + 1, -1), np.asarray(tp, np.float64).reshape(n, L + 1, -1)
    if dc is not None:
        dc, dp = dc.reshape(n, L, dc.shape[-1]), np.asarray(dp, np.float64).reshape(n, L, dc.shape[-1])
    tokens, n_acc, accept, bad, masked = np.full((n, L + 1), -1), np.zeros(n, int), np.zeros((n, L)), 0, 0
    of = lambda c, p, x: float(np.nan_to_num(p[c == x]).sum()) if x >= 0 else 0.0  # noqa: E731
    for b in range(n):
        m = L if lengths is None else min(max(int(lengths[b]), 0), L)
        ref = [tc[b, i, 0] < 0 or (dc is not None and dc[b, i, 0] < 0) for i in range(m)] + [tc[b, m, 0] < 0]
        p = [of(tc[b, i], tp[b, i], drafted[b, i]) for i in range(m)]
        q = [1.0 if dc is None else of(dc[b, i], dp[b, i], drafted[b, i]) for i in range(m)]
        for i in range(m):
            accept[b, i] = np.nan if ref[i] else min(1.0, p[i] / q[i]) if q[i] > 0 else float(p[i] > 0)
        i = 0
        while i < m and not ref[i] and np.float32(ua[b, i]) * np.float32(q[i]) < np.float32(p[i]):
            i += 1
        n_acc[b] = i
        tokens[b, :i] = drafted[b, :i]
        if ref[i]:
            bad += 1
            continue
        full = np.nan_to_num(tp[b, i])
        w = full.copy()
        if i < m:
            for r, c in enumerate(tc[b, i]):
                w[r] -= (1.0 if c == drafted[b, i] else 0.0) if dc is None else of(dc[b, i], dp[b, i], c)
            w = np.maximum(w, 0)
            if w.sum() == 0:
                w = full
        if w.sum() == 0:
            masked += 1
            tokens[b, i] = 0
        else:
            tokens[b, i] = tc[b, i, SR.race(w, ud[b].astype(np.float64))]
    return tokens, n_acc, accept, bad, masked


@pytest.mark.parametrize("n,L,k,dk,V", [(1, 4, 30, 30, 4097), (64, 4, 30, 30, 200), (9, 8, 1, 5, 40), (5, 3, 64, 33, 300),
                                        (3, 2, 65, 200, 500), (2, 64, 30, 30, 100), (4, 0, 30, 1, 100), (3, 2, 1024, 1024, 2000)])
def test_ranked(gpu, n, L, k, dk, V):
    rng = np.random.default_rng([n, L, k, dk])
    tc, tp = ranked_rows(n * (L + 1), k, V, rng)
    dc, dp = ranked_rows(n * L, dk, V, rng, 0.8)
    # half of the drafts' rows near the target's, so that some are accepted
    for r in range(0, n * L, 2):
        m = min(k, dk)
        row = r // L * (L + 1) + r % L
        dc[r, :m] = tc[row, :m]
        rest = np.setdiff1d(np.arange(V), tc[row, :m])[:dk - m]
        dc[r, m:] = rest
        dp[r] = 0
        dp[r, :m] = tp[row, :m] / tp[row, :m].sum()
    drafted = np.array([rng.choice(c, p=p.astype(np.float64) / p.astype(np.float64).sum()) for c, p in zip(dc, dp)],
                       np.int64).reshape(n, L) if n * L else np.zeros((n, L), int)
    u = lambda *s: (rng.integers(0, 1 << 24, s) * 2.0 ** -24).astype(np.float32)  # noqa: E731
    ua, ud = u(n, L), u(n, k)
    lengths = rng.integers(0, L + 1, n) if n > 3 else None
    for certain in (False, True):
        d = (None, None) if certain else (dc, dp)
        got = run_ranked(gpu, tc, tp, *d, drafted, lengths, ua, ud)
        ref = ranked_ref(tc, tp, *d, drafted, lengths, ua, ud)
        assert np.array_equal(got[1], ref[1]) and np.array_equal(got[0], ref[0])
        R.assert_near(got[2], ref[2], 2 * SR.U, "accept")  # one quotient of the given numbers
        assert got[3][0] == ref[3] and got[3][1] == ref[4]


def test_ranked_refused_and_masked_rows(gpu):
    rng = np.random.default_rng(11)
    n, L, k, V = 12, 2, 30, 100
    tc, tp = ranked_rows(n * (L + 1), k, V, rng)
    dc, dp = ranked_rows(n * L, k, V, rng)
    tc3, tp3, dc2, dp2 = tc.reshape(n, L + 1, k), tp.reshape(n, L + 1, k), dc.reshape(n, L, k), dp.reshape(n, L, k)
    drafted = dc2[:, :, 0].astype(np.int64)
    for b in range(n):
        r = b % 6
        if r == 0:
            tc3[b, 0], tp3[b, 0] = -1, np.nan
        elif r == 1:
            tc3[b, L], tp3[b, L] = -1, np.nan
            tc3[b, :L], tp3[b, :L] = dc2[b], dp2[b]
        elif r == 2:
            tc3[b, 1], tp3[b, 1] = np.arange(k), np.nan  # masked
        elif r == 3:
            dc2[b, 1], dp2[b, 1] = -1, np.nan
        elif r == 4:
            dc2[b, 0], dp2[b, 0] = np.arange(k), np.nan
        else:
            drafted[b] = [-1, V + 5]
    u = lambda *s: (rng.integers(0, 1 << 24, s) * 2.0 ** -24).astype(np.float32)  # noqa: E731
    ua, ud = u(n, L), u(n, k)
    got, ref = run_ranked(gpu, tc, tp, dc, dp, drafted, None, ua, ud), ranked_ref(tc, tp, dc, dp, drafted, None, ua, ud)
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])
    assert got[3][0] == ref[3] > 0 and got[3][1] == ref[4]
    R.assert_near(got[2], ref[2], 2 * SR.U, "accept")


@pytest.mark.parametrize("k,top_p", [(30, 0.9), (1, 1.0), (64, 0.7)])
def test_ranked_without_drafts_is_the_samplers_draw(gpu, k, top_p):
    rng = np.random.default_rng([k, 3])
    n, V = 200, 4097
    logits = (rng.standard_normal((n, V)) * 2.5).astype(np.float32)
    u = (rng.integers(1, 1 << 24, (n, k)) * 2.0 ** -24).astype(np.float32)
    s = gpu.sample(logits, u, 0.8, top_p)
    got = run_ranked(gpu, s["cand"], s["probs"], None, None, np.zeros((n, 0), np.int64), None, np.zeros((n, 0)), u)
    assert np.array_equal(got[0][:, 0], s["ids"])


def test_nothing(gpu):
    assert gpu.verify_ranked_raw(4096, 4096, 3, None, None, 0, 0, 0, None, None, None, 4096, 4096, 4096) == 0


def pairs(n, V, td, seed, k):
    """rows of target [n, 2, V] and draft [n, 1, V] alike but for k pairs of places, one of each masked in the one
    and the other in the other, at the same logit: p - q is above 0 at the first of each pair alone.  (Whatever
    order the sums are added in, the pairs' places are beside each other, so that they are the same to the last bit.)"""
    rng = np.random.default_rng([n, V, seed])
    t = np.repeat(rng.standard_normal((n, 1, V)), 2, 1).astype(np.float32) * 2
    d = t[:, :1].copy()
    slots = (V // 2 - 4) // 4
    at = V // 2 // 4 * 4 + 2 * np.sort(rng.permuted(np.tile(np.arange(slots), (n, 1)), axis=1)[:, :k], 1)
    b = np.arange(n)[:, None]
    l = R.to_bits((6 + rng.random((n, k))).astype(np.float32), td)[1]  # noqa: E741
    t[b, 0, at], t[b, 0, at + 1], d[b, 0, at], d[b, 0, at + 1] = l, -np.inf, -np.inf, l
    return t, d, at, np.exp(l), rng


@pytest.mark.parametrize("V", [600, 8192, 9000, 20000, 151936])
@pytest.mark.parametrize("td", ["f32", "bf16"])
def test_rows_alike_but_for_pairs(gpu, V, td):
    """weights that are 0 but at some places, far into the row: with u_draw = 0 the first of them is drawn"""
    n = 48
    for seed, k in enumerate((3, 50, 70)):
        t, d, at, w, rng = pairs(n, V, td, seed, k)
        drafted = at[:, rng.integers(0, k)][:, None] + 1  # p = 0: never accepted
        ud = (rng.integers(0, 1 << 24, n) * 2.0 ** -24).astype(np.float32)
        ud[:n // 2] = 0
        c = w.cumsum(1) / w.sum(1, keepdims=True)
        ud = np.where((np.abs(c - ud[:, None]) < 1e-6).any(1), np.float32(0.0), ud)
        want = at[np.arange(n), (c <= ud[:, None].astype(np.float64)).sum(1)]
        got, _ = run(gpu, t, d, drafted, None, 1.0, 1.0, np.zeros((n, 1)), ud, td, td)
        assert (got[1] == 0).all()
        assert np.array_equal(got[0][:, 0], want), (V, td, seed, got[0][:, 0][got[0][:, 0] != want], want[got[0][:, 0] != want])
        assert (got[0][:, 1] == -1).all() and (got[3][:2] == 0).all()


@pytest.mark.parametrize("V", [20000, 151936])
@pytest.mark.parametrize("rejected", [False, True])
def test_terms_below_the_least_normal_number(gpu, V, rejected):
    """the first half's terms are 2^-1074, which no weight by the sum of twenty ones is: u_draw = 0 draws the first of these"""
    n = 5
    t = np.full((n, 2, V), -np.inf, np.float32)
    t[:, :, :V // 2] = -744.6
    d = np.full((n, 1, V), -np.inf, np.float32)
    d[:, :, 1] = 0.0  # (a token that the target never draws)
    t[:, :, 1] = -np.inf
    ones = V - 20 - 7 * np.arange(n)
    for b in range(n):
        t[b, :, ones[b]:ones[b] + 20] = 0.0
    drafted = np.full((n, 1), 1)
    got, _ = run(gpu, t, d, drafted, None if rejected else np.zeros(n), 1.0, 1.0, np.zeros((n, 1)), np.zeros(n), "f32", "f32")
    assert (got[1] == 0).all() and np.array_equal(got[0][:, 0], ones) and (got[3][:2] == 0).all()


@pytest.mark.parametrize("V", [600, 8192, 9000, 20000, 151936])
def test_rows_alike_but_for_their_last_bits(gpu, V):
    """pairs as above, and between them logits that differ by their last bits, one way or the other: weights
    of 1e-8 of the terms, which sums in 32 bits do not see.  u_draw = 0 draws the first that is above 0 (the sums of both rows
    agree to 1e-9)"""
    n = 48
    for seed, k in enumerate((30, 50, 70)):
        t, d, at, w, rng = pairs(n, V, "f32", seed, k)
        small = (0.25 + 0.25 * rng.random((n, V))).astype(np.float32)
        alike = t[:, 0] == d[:, 0]
        step = rng.choice([-1, 1], (n, V))
        t[:, 0] = np.where(alike, small, t[:, 0])
        d[:, 0] = np.where(alike, (small.view(np.int32) - step).astype(np.int32).view(np.float32), d[:, 0])
        drafted = at[:, rng.integers(0, k)][:, None] + 1
        want = (t[:, 0] > d[:, 0]).argmax(1)
        got, _ = run(gpu, t, d, drafted, None, 1.0, 1.0, np.zeros((n, 1)), np.zeros(n), "f32", "f32")
        assert (got[1] == 0).all() and np.array_equal(got[0][:, 0], want), (V, seed, got[0][:, 0], want)


@pytest.mark.parametrize("u", [0.0, 0.37, 1 - 2.0 ** -24])
def test_sums_that_32_bits_take_amiss(gpu, u):
    """the longest rows of one logit or two, at temperatures whose quotients round apart: the 32-bit sums' quotient is
    2.7e-6 off (each exponent of 13 is 1e-6 off), and the draw's are added again"""
    V = (1 << 24) - 1
    t, d = np.full((1, 2, V), -18.947877883911133, np.float32), np.full((1, 1, V), -18.965412139892578, np.float32)
    t[:, :, :V // 2] = -18.878435134887695
    t[:, :, 7] = d[:, :, 7] = 0.0
    x = V - 9
    t[:, 0, x] = -np.inf
    T, Td, ud = np.float32(1.4257), np.float32(1.4274), np.float32(u)
    got, _ = run(gpu, t, d, np.array([[x]]), None, float(T), float(Td), np.zeros((1, 1)), np.array([ud]), "f32", "f32")
    w = np.maximum(SR.probs(t[0, 0].astype(np.float64), T) - SR.probs(d[0, 0].astype(np.float64), Td), 0)
    assert got[1][0] == 0 and got[0][0, 0] == SR.draw(w, float(ud)) and (got[3][:2] == 0).all()


def test_many_sequences_alike_but_for_pairs(gpu):
    """more sequences of long rows than are split: a workgroup each"""
    n, V, k = 2100, 8200, 40
    t, d, at, w, rng = pairs(n, V, "f32", 1, k)
    drafted = at[:, 5][:, None] + 1
    ud = np.where(np.arange(n) % 2, (rng.integers(0, 1 << 24, n) * 2.0 ** -24), 0.0).astype(np.float32)
    c = w.cumsum(1) / w.sum(1, keepdims=True)
    ud = np.where((np.abs(c - ud[:, None]) < 1e-6).any(1), np.float32(0.0), ud)
    got, _ = run(gpu, t, d, drafted, None, 1.0, 1.0, np.zeros((n, 1)), ud, "f32", "f32")
    assert (got[1] == 0).all() and np.array_equal(got[0][:, 0], at[np.arange(n), (c <= ud[:, None].astype(np.float64)).sum(1)])
