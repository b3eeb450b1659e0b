"""Log probabilities, entropy and alternatives of rows of logits, and their
gradient, against the plain 64-bit form: lengths from one element up, rows cut
into segments, strides and offsets at every element, masks, ties, infinities."""
import math

import numpy as np
import pytest

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


def make(n, V, dtype, seed=0, scale=2.5):
    rng = np.random.default_rng([n, V, seed])
    x = rng.standard_normal((n, V)) * scale
    for r in range(n):
        x[r, rng.integers(0, V, min(V, 5))] += 8
    return rng, *R.to_bits(x, dtype)


def run(gpu, bits, T, banned, tokens, n_top, pad=0, offset=0, use_ws=True, stream=None, entropy=True):
    import hiprt
    n, V = bits.shape
    code = gpu.DTYPE_F32 if bits.dtype == np.float32 else gpu.DTYPE_BF16
    t = tokens.shape[1]
    with R.Arena() as D:
        flat = R.with_stride(bits, V + pad, offset, 0x7f80 if code else np.inf)  # what lies between rows must not matter
        lg = D.put(flat)
        lp, H, st = D.room(4 * n * t, 0xee), D.room(4 * n, 0xee), D.room(8 * n, 0xee)
        ids, tlp, cnt = D.room(4 * n * n_top, 0xee), D.room(4 * n * n_top, 0xee), D.room(16, 0)
        tok = D.put(tokens.astype(np.int32))
        temp = ("ptr", D.put(np.asarray(T, np.float32)).ptr) if np.ndim(T) else float(T)
        ban = D.put(np.asarray(banned, np.int32)).ptr if banned is not None else None
        ws = None
        if use_ws:
            need = gpu.lib().d3s_logprob_workspace_bytes(code, n, V, n_top)
            W = gpu.Workspace(need)
            D.held.append(W.buf)
            ws = W.arg()
        rc = gpu.logprob_raw(lg.ptr + offset * bits.itemsize, code, n, V, V + pad, temp, ban, tok.ptr, t, lp.ptr,
                             H.ptr if entropy else None, st.ptr, n_top, ids.ptr, tlp.ptr, cnt.ptr, workspace=ws,
                             stream=stream.ptr if stream else None)
        assert rc == 0
        hiprt.synchronize()
        return dict(logprobs=lp.download((n, t), np.float32), H=H.download((n,), np.float32),
                    stats=st.download((n, 2), np.float32), top_ids=ids.download((n, n_top), np.int32),
                    top_logprobs=tlp.download((n, n_top), np.float32), counters=cnt.download((4,), np.uint32))


def check(got, ref, entropy=True):
    R.assert_near(got["logprobs"], ref["logprobs"], R.score_tol(ref, ref["logprobs"]), "logprobs")
    if entropy:
        R.assert_near(got["H"], ref["H"], R.entropy_tol(ref), "entropy")
    R.assert_near(got["stats"][:, 0], ref["m"], 0, "greatest")
    R.assert_near(got["stats"][:, 1], ref["logS"], R.score_tol(ref, ref["logS"][:, None])[:, 0], "log sum")
    assert np.array_equal(got["top_ids"], ref["top_ids"])
    R.assert_near(got["top_logprobs"], ref["top_logprobs"], R.score_tol(ref, ref["top_logprobs"]), "alternatives")
    assert got["counters"].tolist() == [int(ref["refused"].sum()), int(ref["masked"].sum()), 0, 0]


def temperatures(T, n):
    return np.asarray(np.broadcast_to(np.float32(T), n), np.float64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,V,t,top,pad,offset", [
    (1, 1, 1, 1, 0, 0), (3, 2, 2, 2, 1, 1), (5, 7, 1, 7, 0, 3), (2, 63, 4, 5, 5, 0), (9, 64, 1, 64, 0, 0),
    (4, 255, 1, 20, 2, 7), (7, 1000, 3, 64, 3, 1), (1, 4097, 1, 5, 0, 0), (300, 4097, 1, 0, 7, 2), (9, 4096, 64, 10, 0, 0),
    (3, 8191, 1, 64, 0, 5), (1, 16384, 1, 20, 0, 1), (2, 50001, 2, 33, 1, 0), (5, 151936, 1, 20, 0, 0),
    (1, 151936, 1, 64, 0, 3), (1030, 9001, 1, 1, 0, 0), (1, 1000003, 1, 7, 0, 1)])
def test_rows(gpu, n, V, t, top, pad, offset, dtype):
    rng, bits, l = make(n, V, dtype)
    tokens = rng.integers(-1, V + 1, (n, t))  # some are none
    got = run(gpu, bits, 0.7, None, tokens, top, pad, offset)
    check(got, R.score(l, temperatures(0.7, n), None, tokens, top))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [50, 4097, 40001])
def test_temperatures_and_banned(gpu, V, dtype):
    n = 8
    rng, bits, l = make(n, V, dtype, 1)
    T = np.array([0.0, -3.0, 1e-5, 0.05, 0.7, 1.0, 30.0, 1e6], np.float32)
    banned = np.array([0, -1, V - 1, V, 3, l[5].argmax(), -7, 1 << 30])
    tokens = rng.integers(0, V, (n, 2))
    tokens[4, 0] = 3  # a banned token
    got = run(gpu, bits, T, banned, tokens, 10)
    check(got, R.score(l, T.astype(np.float64), banned, tokens, 10))


@pytest.mark.parametrize("V", [1, 40, 4097, 40001])
def test_refused_and_masked_rows(gpu, V):
    n = 7
    rng, bits, l = make(n, V, "f32", 2)
    l = l.astype(np.float32)
    l[0, V // 2] = np.nan
    l[1, V - 1] = np.inf
    l[2] = -np.inf
    l[3] = -np.inf
    l[3, V // 3] = -5.0  # one place left
    l[4, 0] = -np.inf
    T = np.array([1, 1, 1, 1, 1, np.inf, np.nan], np.float32)
    tokens = np.stack([rng.integers(0, V, n), np.full(n, -1)], 1)
    tokens[3, 0] = V // 3
    top = min(V, 9)
    got = run(gpu, l, T, None, tokens, top)
    check(got, R.score(l.astype(np.float64), T.astype(np.float64), None, tokens, top))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lowest_values_and_huge_logits(gpu, dtype):
    """masks of the type's lowest value, rows of nothing else, logits whose
    quotient by T overflows, and shifts far from the logits' spread"""
    n, V = 6, 5000
    rng, bits, l = make(n, V, dtype, 3)
    low = float(np.float32(-3.3895314e38))  # bf16's lowest
    l = l.astype(np.float32)
    l[0, 10:] = low
    l[1] = low
    l[2] = low
    l[2, 77] = -low
    l[3] = np.where(rng.random(V) < 0.5, low, l[3])
    l[4] += 1e4
    l[5] *= 1e30
    T = np.array([1, 1, 1, 1e-5, 1e-5, 1e-5], np.float32)
    bits, l = R.to_bits(l, dtype)
    tokens = np.stack([rng.integers(0, V, n), l.argmax(1)], 1)
    got = run(gpu, bits, T, None, tokens, 20)
    check(got, R.score(l, T.astype(np.float64), None, tokens, 20))


@pytest.mark.parametrize("V", [5, 1500, 4097, 70001])
def test_ties(gpu, V):
    """equal rows, two values, zeros of both signs: the lowest indices first"""
    n = 4
    rng = np.random.default_rng(4)
    l = np.zeros((n, V), np.float32)
    l[1] = rng.integers(0, 2, V)
    l[2] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    l[3] = np.round(rng.standard_normal(V) * 2)
    top = min(64, V)
    tokens = rng.integers(0, V, (n, 1))
    for dtype in ("f32", "bf16"):
        bits, ld = R.to_bits(l, dtype)
        check(run(gpu, bits, 1.0, None, tokens, top), R.score(ld, np.ones(n), None, tokens, top))


def test_without_workspace_and_entropy_and_on_a_stream(gpu):
    import hiprt
    rng, bits, l = make(3, 60000, "bf16", 5)
    tokens = rng.integers(0, 60000, (3, 1))
    ref = R.score(l, temperatures(0.9, 3), None, tokens, 4)
    a = run(gpu, bits, 0.9, None, tokens, 4)
    s = hiprt.Stream()
    b = run(gpu, bits, 0.9, None, tokens, 4, use_ws=False, stream=s)
    check(b, ref)
    for name in a:
        assert np.array_equal(a[name], b[name], equal_nan=True)
    c = run(gpu, bits, 0.9, None, tokens, 4, use_ws=False, stream=s, entropy=False)
    check(c, ref, entropy=False)
    assert gpu.lib().d3s_stream_workspace_release(s.ptr) == 0
    s.destroy()


def test_captured_and_replayed(gpu):
    """one workspace, a graph of two calls replayed with other work between"""
    import ctypes

    import hiprt
    n, V, top = 2, 40000, 8
    H = hiprt.hip()
    s = hiprt.Stream()
    rng, bits, _ = make(n, V, "bf16", 6)
    tokens = rng.integers(0, V, (n, 1))
    with R.Arena() as D:
        lg, tok = D.put(bits), D.put(tokens.astype(np.int32))
        lp, ent, st, grad = D.room(4 * n), D.room(4 * n), D.room(8 * n), D.room(2 * n * V)
        ids, g = D.room(4 * n * top), D.put(np.ones((n, 1), np.float32))
        W = gpu.Workspace(gpu.lib().d3s_logprob_workspace_bytes(1, n, V, top))
        D.held.append(W.buf)
        hiprt.synchronize()

        def call(ws):
            rc = gpu.logprob_raw(lg.ptr, 1, n, V, V, 1.0, None, tok.ptr, 1, lp.ptr, ent.ptr, st.ptr, top, ids.ptr,
                                 workspace=ws, stream=s.ptr)
            return rc or gpu.logprob_backward_raw(lg.ptr, 1, n, V, V, 1.0, None, tok.ptr, 1, st.ptr, ent.ptr, g.ptr, None,
                                                  grad.ptr, V, stream=s.ptr)

        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        hiprt.check(H.hipStreamBeginCapture(s.ptr, 2))
        refused = call(None)  # without a workspace of the caller's: nothing is recorded
        rc = call(W.arg())
        hiprt.check(H.hipStreamEndCapture(s.ptr, ctypes.byref(graph)))
        assert refused == -7 and rc == 0
        assert hiprt.graph_node_types(graph) == ["kernel", "kernel"]
        hiprt.check(H.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0))
        for i in range(4):
            bits, l = R.to_bits(rng.standard_normal((n, V)) * 3, "bf16")
            lg.upload(bits)
            hiprt.synchronize()
            hiprt.check(H.hipGraphLaunch(ex, s.ptr))
            s.synchronize()
            ref = R.score(l, np.ones(n), None, tokens, top)
            R.assert_near(lp.download((n, 1), np.float32), ref["logprobs"], R.score_tol(ref, ref["logprobs"]))
            assert np.array_equal(ids.download((n, top), np.int32), ref["top_ids"])
            dx, err = R.score_grad(ref, tokens, np.ones((n, 1)), None)
            R.assert_near(R.from_bits(grad.download((n, V), np.uint16)), dx, err * 4 + R.BF16 * np.abs(dx))
            assert call(W.arg()) == 0  # eager work on the same workspace between replays
            s.synchronize()
        H.hipGraphExecDestroy(ex)
        H.hipGraphDestroy(graph)
        s.destroy()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_32_bits(gpu, dtype):
    """the second row starts past 2^31 elements (2^32 bytes and more)"""
    import hiprt
    V, stride = 3000, (1 << 31) + 24
    rng, bits, l = make(2, V, dtype, 7)
    code = gpu.DTYPE_F32 if dtype == "f32" else gpu.DTYPE_BF16
    tokens = rng.integers(0, V, (2, 1))
    with R.Arena() as D:
        big = D.room((stride + V) * bits.itemsize)
        big.upload(bits[0]).upload(bits[1], stride * bits.itemsize)
        lp, ent, st, tok = D.room(8), D.room(8), D.room(16), D.put(tokens.astype(np.int32))
        g = D.put(np.ones((2, 1), np.float32))
        assert gpu.logprob_raw(big.ptr, code, 2, V, stride, 1.0, None, tok.ptr, 1, lp.ptr, ent.ptr, st.ptr) == 0
        hiprt.synchronize()
        ref = R.score(l, np.ones(2), None, tokens, 0)
        R.assert_near(lp.download((2, 1), np.float32), ref["logprobs"], R.score_tol(ref, ref["logprobs"]))
        assert gpu.logprob_backward_raw(big.ptr, code, 2, V, stride, 1.0, None, tok.ptr, 1, st.ptr, ent.ptr, g.ptr, None,
                                        big.ptr, stride) == 0
        hiprt.synchronize()
        dx, err = R.score_grad(ref, tokens, np.ones((2, 1)), None)
        for r in range(2):
            got = R.from_bits(big.download((V,), bits.dtype, r * stride * bits.itemsize))
            R.assert_near(got, dx[r], err[r] * 4 + (R.BF16 * np.abs(dx[r]) if dtype == "bf16" else 0))


# ---- the gradient ----
def run_grad(gpu, bits, T, banned, tokens, ref, g, gH, pad=0, grad_pad=0, grad_offset=0, in_place=False):
    import hiprt
    n, V = bits.shape
    es = bits.itemsize
    code = gpu.DTYPE_F32 if bits.dtype == np.float32 else gpu.DTYPE_BF16
    with R.Arena() as D:
        lg = D.put(R.with_stride(bits, V + pad, grad_offset, 0x7f80 if code else np.inf))
        size = grad_offset + (n - 1) * (V + grad_pad) + V + 16
        out = lg if in_place else D.room(size * es, 0x5a)
        stats = np.stack([ref["m"], ref["logS"]], 1).astype(np.float32)
        temp = ("ptr", D.put(np.asarray(T, np.float32)).ptr)
        rc = gpu.logprob_backward_raw(
            lg.ptr + grad_offset * es, code, n, V, V + pad, temp,
            D.put(np.asarray(banned, np.int32)).ptr if banned is not None else None, D.put(tokens.astype(np.int32)).ptr,
            tokens.shape[1], D.put(stats).ptr, D.put(ref["H"].astype(np.float32)).ptr if gH is not None else None,
            D.put(g.astype(np.float32)).ptr, D.put(gH.astype(np.float32)).ptr if gH is not None else None,
            out.ptr + grad_offset * es, V + (pad if in_place else grad_pad))
        assert rc == 0
        hiprt.synchronize()
        if in_place:
            flat = out.download((grad_offset + (n - 1) * (V + pad) + V,), bits.dtype)
            return R.rows_at(flat, n, V, V + pad, grad_offset)
        flat = out.download((size,), bits.dtype)
        inside = np.zeros(size, bool)
        for r in range(n):
            inside[grad_offset + r * (V + grad_pad): grad_offset + r * (V + grad_pad) + V] = True
        assert (flat[~inside].view(np.uint8) == 0x5a).all(), "written outside the rows"
        return R.rows_at(flat, n, V, V + grad_pad, grad_offset)


def check_grad(got, dx, err):
    tol = err + (R.BF16 * np.abs(dx) if got.dtype == np.uint16 else R.U * np.abs(dx))
    R.assert_near(R.from_bits(got), dx, tol, "gradient")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,V,t,pad,grad_pad,offset", [
    (1, 1, 1, 0, 0, 0), (3, 2, 2, 1, 0, 1), (4, 9, 1, 0, 3, 2), (5, 64, 64, 0, 0, 0), (2, 1000, 3, 5, 0, 1),
    (40, 4097, 1, 0, 0, 0), (9, 4097, 1, 7, 0, 0), (3, 4097, 4, 0, 7, 3), (2, 151936, 1, 0, 0, 0), (1, 300007, 2, 1, 0, 5)])
def test_gradient(gpu, n, V, t, pad, grad_pad, offset, dtype):
    rng, bits, l = make(n, V, dtype, 8)
    T = rng.uniform(0.4, 1.5, n).astype(np.float32)
    tokens = rng.integers(-1, V + 1, (n, t))
    tokens[0, -1] = tokens[0, 0]  # given twice
    banned = np.where(rng.random(n) < 0.5, rng.integers(0, V, n), -1) if V > 2 else None
    g, gH = rng.standard_normal((n, t)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    ref = R.score(l, T.astype(np.float64), banned, tokens, 0)
    for h in (gH, None):
        dx, err = R.score_grad(ref, tokens, g.astype(np.float64), h)
        check_grad(run_grad(gpu, bits, T, banned, tokens, ref, g, h, pad, grad_pad, offset), dx, err)
        check_grad(run_grad(gpu, bits, T, banned, tokens, ref, g, h, pad, 0, offset, in_place=True), dx, err)


def test_gradient_of_odd_rows(gpu):
    """masked places, one place left, all masked, refused, and rows without a gradient"""
    n, V = 8, 3001
    rng, bits, l = make(n, V, "f32", 9)
    l = l.astype(np.float32)
    l[0, rng.random(V) < 0.5] = -np.inf
    l[1] = -np.inf
    l[1, 5] = 2.0
    l[2] = -np.inf
    l[3, 9] = np.nan
    l[4, 9] = np.nan
    l[5, 100:] = np.float32(-3.4028235e38)
    l[6] = np.float32(-3.4028235e38)
    T = np.array([1, 1, 1, 1, 1, 1, 1, np.inf], np.float32)
    tokens = rng.integers(0, V, (n, 1))
    tokens[1, 0] = 5
    g = rng.standard_normal((n, 1)).astype(np.float32)
    gH = rng.standard_normal(n).astype(np.float32)
    g[4], gH[4] = 0, 0
    ref = R.score(l.astype(np.float64), T.astype(np.float64), None, tokens, 0)
    dx, err = R.score_grad(ref, tokens, g.astype(np.float64), gH)
    dx[4] = 0  # refused, but without a gradient
    err[4] = 0
    dx[3], dx[7] = np.nan, np.nan
    check_grad(run_grad(gpu, l, T, None, tokens, ref, g, gH), dx, np.nan_to_num(err, nan=0.0) + 1e-37)


def test_gradient_against_differences(gpu):
    """central differences of the forward kernel's own outputs: their error is a
    third derivative's, h^2 / 6 times at most 2, and the outputs' rounding over 2 h"""
    n, V, h = 2, 12, 1 / 64
    rng, bits, l = make(n, V, "f32", 10, scale=1.0)
    l = np.float32(rng.integers(-64, 64, (n, V)) / 32)  # l + h is exact
    tokens = rng.integers(0, V, (n, 2))
    g, gH = rng.standard_normal((n, 2)).astype(np.float32), rng.standard_normal(n).astype(np.float32)

    def loss(x):
        o = run(gpu, x, 1.0, None, tokens, 0)
        return (o["logprobs"].astype(np.float64) * g).sum(1) + o["H"].astype(np.float64) * gH

    ref = R.score(l.astype(np.float64), np.ones(n), None, tokens, 0)
    got = run_grad(gpu, l, np.ones(n), None, tokens, ref, g, gH)
    for j in range(V):
        up, down = l.copy(), l.copy()
        up[:, j] += np.float32(h)
        down[:, j] -= np.float32(h)
        d = (loss(up) - loss(down)) / (2 * h)
        size = np.abs(g).sum(1) + np.abs(gH) * 8
        assert (np.abs(d - got[:, j]) <= size * (h * h + 64 * R.U / h)).all(), j
