"""Dense layers with their epilogue, both operand orders, and the epilogue's
gradient, against 64 bits: sizes from one up, edges of every tile, strides and
addresses at every element, activations, kept pre-activations, sums in place."""
import numpy as np
import pytest

import train_ref as R

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


def product(gpu, m, n, k, xt=False, wt=False, act="none", bias=False, residual=False, keep=False, out="bf16", pads=(0, 0, 0),
            offset=0, in_place=False, seed=0, scale=1.0):
    """runs the call and checks it whole"""
    import hiprt
    rng = np.random.default_rng([m, n, k, seed])
    xs, ws = ((k, m) if xt else (m, k)), ((k, n) if wt else (n, k))
    xb, x = R.to_bits(rng.standard_normal(xs) * scale, "bf16")
    wb, w = R.to_bits(rng.standard_normal(ws) * max(k, 1) ** -0.5, "bf16")
    x, w = x.T if xt else x, w.T if wt else w
    b, bv = R.to_bits(rng.standard_normal(n), "bf16")
    r, rv = R.to_bits(rng.standard_normal((m, n)), out)
    es = 4 if out == "f32" else 2
    ystride = n + pads[2]
    with R.Arena() as D:
        # NaN between the rows and before them: reading it into a sum would show
        dx = D.put(R.with_stride(xb, xs[1] + pads[0], offset, 0x7fc0))
        dw = D.put(R.with_stride(wb, ws[1] + pads[1], offset, 0x7fc0))
        size = offset + (m - 1) * ystride + n + 8
        y = D.room(size * es, 0x5a)
        z = D.room(size * 2, 0x5a)
        if in_place:
            flat = y.download((size,), r.dtype)
            for i in range(m):
                flat[offset + i * ystride: offset + i * ystride + n] = r[i]
            y.upload(flat)
        res = None
        if residual:
            res = y.ptr + offset * es if in_place else D.put(R.with_stride(r, n + 3, offset, 0)).ptr + offset * es
        rc = gpu.dense_raw(dx.ptr + 2 * offset, xs[1] + pads[0], dw.ptr + 2 * offset, ws[1] + pads[1], m, n, k,
                           y.ptr + offset * es, ystride, gpu.DTYPE_F32 if out == "f32" else gpu.DTYPE_BF16,
                           x_transposed=xt, w_transposed=wt, bias=D.put(b).ptr if bias else None,
                           activation=gpu.ACTIVATIONS[act], residual=res, residual_stride=ystride if in_place else n + 3,
                           z=z.ptr + 2 * offset if keep else None, z_stride=ystride)
        assert rc == 0
        hiprt.synchronize()
        fy, fz = y.download((size,), r.dtype), z.download((size,), np.uint16)
    inside = np.zeros(size, bool)
    for i in range(m):
        inside[offset + i * ystride: offset + i * ystride + n] = True
    assert (fy[~inside].view(np.uint8) == 0x5a).all(), "y written outside"
    assert (fz[~inside if keep else slice(None)].view(np.uint8) == 0x5a).all(), "z written outside"
    zr = x @ w.T
    # fp32 sums of exact products in some order (a step of 2 u an addition covers truncation in the matrix cores)
    err = 2 * R.U * k * (np.abs(x) @ np.abs(w).T)
    if bias:
        zr = zr + bv
        err = err + R.U * np.abs(zr)
    if keep:
        R.assert_near(R.from_bits(R.rows_at(fz, m, n, ystride, offset)), zr, err + R.BF16 * (np.abs(zr) + err), "z")
    yr = R.act(zr, act)
    if act != "none":
        # slopes are at most 1.13; the functions take fewer than 16 roundings relative to z
        err = 1.13 * err + 16 * R.U * np.abs(zr)
    if residual:
        yr = yr + rv
        err = err + R.U * np.abs(yr)
    tol = err + (R.BF16 * (np.abs(yr) + err) if out == "bf16" else R.U * np.abs(yr))
    R.assert_near(R.from_bits(R.rows_at(fy, m, n, ystride, offset)), yr, tol + 1e-38, "y")


ORDERS = [(False, False), (False, True), (True, False), (True, True)]


@pytest.mark.parametrize("xt,wt", ORDERS)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 4, 8), (2, 3, 5), (7, 16, 33), (16, 17, 64), (63, 65, 31), (128, 128, 32), (129, 127, 100), (5, 300, 257),
    (200, 1, 70), (1, 2048, 2048), (64, 513, 130), (257, 260, 96), (300, 40, 1000)])
def test_sizes(gpu, m, n, k, xt, wt):
    product(gpu, m, n, k, xt, wt)
    product(gpu, m, n, k, xt, wt, bias=True, residual=True, out="f32", pads=(1, 3, 1), offset=1)


@pytest.mark.parametrize("xt,wt", ORDERS)
@pytest.mark.parametrize("m,n,k", [(256, 256, 64), (256, 256, 128), (512, 768, 256), (300, 520, 192), (1024, 257, 320),
                                   (513, 1000, 328), (260, 4097, 264), (2048, 512, 1031)])
def test_large_tiles(gpu, m, n, k, xt, wt):
    """whole and cut tiles of the large products, rows at 16 bytes and off them"""
    product(gpu, m, n, k, xt, wt, bias=True, act="silu", keep=True)
    product(gpu, m, n, k, xt, wt, out="f32", residual=True, pads=(8 - xt * m % 8, 8 - wt * n % 8, 0))
    product(gpu, m, n, k, xt, wt, pads=(-(m if xt else k) % 8, -(n if wt else k) % 8, 5), residual=True, act="gelu")
    product(gpu, m, n, k, xt, wt, pads=(3, 0, 0), offset=3)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 100, 256), (40, 130, 72), (384, 512, 128)])
def test_epilogue(gpu, act, out, m, n, k):
    for bias, residual, keep in [(True, True, True), (False, True, False), (True, False, False), (False, False, True)]:
        product(gpu, m, n, k, act=act, out=out, bias=bias, residual=residual, keep=keep, scale=4.0)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])
@pytest.mark.parametrize("n,k", [(2048, 2048), (4097, 512), (100, 1024), (33, 4104)])
def test_few_rows(gpu, m, n, k):
    product(gpu, m, n, k, bias=True, act="silu", residual=True)
    product(gpu, m, n, k, out="f32", pads=(8, 8, 1))


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (30, 50, 40), (300, 600, 128)])
def test_added_in_place(gpu, m, n, k, out):
    product(gpu, m, n, k, residual=True, out=out, in_place=True)
    product(gpu, m, n, k, True, True, residual=True, out=out, in_place=True, pads=(0, 0, 5))


def test_nothing_summed(gpu):
    for m in (1, 70, 300):
        product(gpu, m, 33, 0, bias=True, residual=True, act="gelu")
        product(gpu, m, 300, 0)


def test_long_sums(gpu):
    product(gpu, 64, 128, 20000, True, True, out="f32")
    product(gpu, 256, 256, 16384, True, True, out="f32")
    product(gpu, 3, 40, 65536)


def test_infinities_stay_in_their_rows(gpu):
    """a row of x with an infinity and a NaN, an output of w with one: no other output sees them"""
    import hiprt
    m, n, k = 300, 300, 192
    rng = np.random.default_rng(1)
    xb, x = R.to_bits(rng.standard_normal((m, k)), "bf16")
    wb, w = R.to_bits(rng.standard_normal((n, k)), "bf16")
    xb[7, 3], xb[299, 191], wb[64, 0] = 0x7f80, 0x7fc0, 0xff80
    with R.Arena() as D:
        y = D.room(2 * m * n)
        assert gpu.dense_raw(D.put(xb).ptr, k, D.put(wb).ptr, k, m, n, k, y.ptr, n, gpu.DTYPE_BF16) == 0
        hiprt.synchronize()
        got = R.from_bits(y.download((m, n), np.uint16))
    odd = np.zeros((m, n), bool)
    odd[7], odd[299], odd[:, 64] = True, True, True
    assert np.isfinite(got[~odd]).all() and not np.isfinite(got[odd]).any()


@pytest.mark.parametrize("m", [2, 300])
def test_rows_past_32_bits(gpu, m):
    """x's last row lies past 2^31 elements"""
    import hiprt
    n, k = 40, 64
    stride = ((1 << 31) // (m - 1) + 64) // 8 * 8
    rng = np.random.default_rng(2)
    xb, x = R.to_bits(rng.standard_normal((m, k)), "bf16")
    wb, w = R.to_bits(rng.standard_normal((n, k)), "bf16")
    with R.Arena() as D:
        big = D.room(2 * ((m - 1) * stride + k))
        for i in range(m):
            big.upload(xb[i], 2 * i * stride)
        y = D.room(4 * m * n)
        assert gpu.dense_raw(big.ptr, stride, D.put(wb).ptr, k, m, n, k, y.ptr, n, gpu.DTYPE_F32) == 0
        hiprt.synchronize()
        R.assert_near(y.download((m, n), np.float32), x @ w.T, 2 * R.U * k * (np.abs(x) @ np.abs(w).T))


def test_gradients_against_differences(gpu):
    """dx and dw of sum(g * y) by the same call with operands transposed, against
    differences of the call's own fp32 outputs: y is linear in x and w, so only
    roundings remain (k products of at most size ~16, over the step)"""
    import hiprt
    m, n, k = 6, 10, 24
    rng = np.random.default_rng(3)
    ints = lambda *s: R.to_bits(rng.integers(-4, 5, s), "bf16")  # noqa: E731  (every sum is exact)
    (xb, x), (wb, w), (gb, g) = ints(m, k), ints(n, k), ints(m, n)

    def call(a, b, m, n, k, **kw):
        with R.Arena() as D:
            y = D.room(4 * m * n)
            assert gpu.dense_raw(D.put(a).ptr, a.shape[1], D.put(b).ptr, b.shape[1], m, n, k, y.ptr, n, gpu.DTYPE_F32, **kw) == 0
            hiprt.synchronize()
            return y.download((m, n), np.float32).astype(np.float64)

    dx = call(gb, wb, m, k, n, w_transposed=True)
    dw = call(gb, xb, n, k, m, x_transposed=True, w_transposed=True)
    loss = lambda a, b: (call(a, b, m, n, k) * g).sum()  # noqa: E731
    for i, j in [(0, 0), (5, 23), (3, 7)]:
        up = x.copy()
        up[i, j] += 1
        assert loss(R.to_bits(up, "bf16")[0], wb) - loss(xb, wb) == dx[i, j]
    for i, j in [(0, 0), (9, 23), (4, 11)]:
        up = w.copy()
        up[i, j] += 1
        assert loss(xb, R.to_bits(up, "bf16")[0]) - loss(xb, wb) == dw[i, j]


# ---- the epilogue's gradient ----
def slopes(gpu, m, n, act, dbias=True, dz=True, pads=(0, 0, 0), offset=0, in_place=False, scale=2.0):
    import hiprt
    rng = np.random.default_rng([m, n])
    db, d = R.to_bits(rng.standard_normal((m, n)), "bf16")
    zb, z = R.to_bits(rng.standard_normal((m, n)) * scale, "bf16")
    with R.Arena() as D:
        dy = D.put(np.concatenate([R.with_stride(db, n + pads[0], offset, 0x7fc0), np.full(8, 0x7fc0, np.uint16)]))
        zz = D.put(np.concatenate([R.with_stride(zb, n + pads[1], offset, 0x7fc0), np.full(8, 0x7fc0, np.uint16)]))
        size = offset + (m - 1) * (n + pads[2]) + n + 8 if m else 8
        out, sums = (dy if in_place else D.room(2 * size, 0x5a)), D.room(4 * n + 16, 0x5a)
        rc = gpu.dense_activation_backward_raw(dy.ptr + 2 * offset, n + pads[0], zz.ptr + 2 * offset if act != "none" else None,
                                               n + pads[1], m, n, gpu.ACTIVATIONS[act], out.ptr + 2 * offset if dz else None,
                                               n + pads[0 if in_place else 2], sums.ptr if dbias else None)
        assert rc == 0
        hiprt.synchronize()
        fs = sums.download((n + 4,), np.float32)
        fo = out.download((out.nbytes // 2,), np.uint16)
    stride = n + pads[0 if in_place else 2]
    v = d * R.slope(z, act)
    # the slope's functions: fewer than 16 roundings relative to (1 + |z|)
    err = 16 * R.U * np.abs(d) * (1 + np.abs(z)) if act != "none" else np.zeros_like(v)
    if dz:
        R.assert_near(R.from_bits(R.rows_at(fo, m, n, stride, offset)), v, err + R.BF16 * (np.abs(v) + err) + 1e-39, "dz")
        if not in_place:
            inside = np.zeros(fo.size, bool)
            for i in range(m):
                inside[offset + i * stride: offset + i * stride + n] = True
            assert (fo[~inside].view(np.uint8) == 0x5a).all()
    if dbias:
        R.assert_near(fs[:n], v.sum(0), err.sum(0) + R.U * (m + 1) * np.abs(v).sum(0) + 1e-38, "dbias")
        assert (fs[n:].view(np.uint8) == 0x5a).all()
    else:
        assert (fs.view(np.uint8) == 0x5a).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(1, 1), (3, 7), (100, 8), (33, 9), (64, 512), (1000, 513), (5, 4097), (4100, 40), (700, 2048)])
def test_activation_backward(gpu, m, n, act):
    slopes(gpu, m, n, act)
    slopes(gpu, m, n, act, pads=(1, 5, 3), offset=1, scale=6.0)
    slopes(gpu, m, n, act, in_place=True, pads=(2, 0, 0))


def test_activation_backward_parts(gpu):
    slopes(gpu, 50, 70, "silu", dbias=False)
    slopes(gpu, 50, 70, "silu", dz=False)
    slopes(gpu, 50, 70, "none", dz=False)
    slopes(gpu, 0, 70, "none")


def test_activation_backward_far_values(gpu):
    """slopes at the ends: 0 and 1, no NaN from exponentials that overflow"""
    import hiprt
    z = np.float32([-1e30, -300, -100, -90, -20, -0.0, 0.0, 20, 90, 100, 300, 1e30])
    zb, zv = R.to_bits(z, "bf16")
    n = z.size
    for act in ACTS[1:]:
        with R.Arena() as D:
            out = D.room(2 * n)
            one = D.put(R.to_bits(np.ones(n), "bf16")[0])
            assert gpu.dense_activation_backward_raw(one.ptr, n, D.put(zb).ptr, n, 1, n, gpu.ACTIVATIONS[act], out.ptr, n, None) == 0
            hiprt.synchronize()
            got = R.from_bits(out.download((n,), np.uint16))
        with np.errstate(all="ignore"):
            ref = np.where(zv > 50, 1.0, np.where(zv < -50, 0.0, R.slope(np.clip(zv, -50, 50), act)))
        R.assert_near(got, ref, R.BF16 * np.abs(ref) + 1e-6, act)
