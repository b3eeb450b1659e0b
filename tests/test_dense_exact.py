"""Dense layers of small whole numbers: every product and every partial sum is a
whole number below 2^24, so the fp32 result is the exact one in whatever order it
is summed, and a single inner index left out or taken twice shows at any length."""
import numpy as np
import pytest

import train_ref as R
from test_train_paths import SPLIT

pytestmark = pytest.mark.gpu

ORDERS = [(False, False), (False, True), (True, False), (True, True)]
VALUES = np.arange(-2, 3, dtype=np.float32)
BITS, _ = R.to_bits(VALUES, "bf16")


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


def whole_numbers(rng, rows, columns):
    """(bf16 bits, fp32 values) of -2 .. 2"""
    i = rng.integers(0, 5, (rows, columns), np.uint8)
    return BITS[i], VALUES[i]


def product(gpu, m, n, k, xt=False, wt=False, pads=(0, 0, 0), offset=0, added=False, seed=0):
    """y = x w^T (+ y): every output equal to the exact one, and nothing else written"""
    import hiprt
    rng = np.random.default_rng([m, n, k, seed])
    xs, ws = ((k, m) if xt else (m, k)), ((k, n) if wt else (n, k))
    (xb, x), (wb, w) = whole_numbers(rng, *xs), whole_numbers(rng, *ws)
    stride = n + pads[2]
    size = offset + (m - 1) * stride + n + 8
    before = np.full(size, 7.0, np.float32)
    inside = np.zeros(size, bool)
    for i in range(m):
        inside[offset + i * stride: offset + i * stride + n] = True
    if added:
        before[inside] = rng.integers(-1000, 1000, m * n)
    want = before.copy()
    # (fp32 is exact here too: |sums| <= 4 k + 1000 < 2^24)
    want[inside] = ((x.T if xt else x) @ (w if wt else w.T)).reshape(-1) + (before[inside] if added else 0)
    with R.Arena() as D:
        dx = D.put(R.with_stride(xb, xs[1] + pads[0], offset, 0x7fc0))
        dw = D.put(R.with_stride(wb, ws[1] + pads[1], offset, 0x7fc0))
        y = D.put(before)
        at = y.ptr + 4 * offset
        assert gpu.dense_raw(dx.ptr + 2 * offset, xs[1] + pads[0], dw.ptr + 2 * offset, ws[1] + pads[1], m, n, k, at, stride,
                             gpu.DTYPE_F32, x_transposed=xt, w_transposed=wt, residual=at if added else None,
                             residual_stride=stride) == 0
        hiprt.synchronize()
        got = y.download((size,), np.float32)
    bad = np.flatnonzero(got != want)
    assert bad.size == 0, (m, n, k, bad.size, bad[:4], got[bad[:4]], want[bad[:4]])


@pytest.mark.parametrize("xt,wt", ORDERS)
@pytest.mark.parametrize("m,n", [(3, 40), (20, 100), (60, 100), (130, 200), (257, 70)])
def test_long_inner_lengths(gpu, m, n, xt, wt):
    """around whole stages, whole batches of the kernel of few rows, and the shares of
    two to sixteen splits"""
    for k in (1023, 1024, 1025, 1536, 1599, 2047, 2049, 2111, 2561, 3000, 3073, 4095, 4097, 5121, 6000, 8191, 8193, 8255,
              16383, 16385, 20000, 65537):
        product(gpu, m, n, k, xt, wt)
    for k in (1025, 3073, 8193, 20011):
        product(gpu, m, n, k, xt, wt, pads=(3, 1, 2), offset=1, added=True)
        product(gpu, m, n, k, xt, wt, pads=(-(m if xt else k) % 8, -(n if wt else k) % 8, 0), added=True)


@pytest.mark.parametrize("shape", SPLIT)
def test_split_sums(gpu, shape):
    product(gpu, *shape)
    product(gpu, *shape, added=True, pads=(8, 8, 1))


@pytest.mark.parametrize("xt,wt", ORDERS)
@pytest.mark.parametrize("m,n", [(256, 2048), (2304, 2304), (2049, 2070), (1500, 11008), (11008, 1500)])
def test_stages_of_large_outputs(gpu, m, n, xt, wt):
    """several rounds of tiles, rows or outputs peeled off them, a last round apart"""
    for k in (64, 65, 127, 192, 321):
        product(gpu, m, n, k, xt, wt, added=k == 321)
    product(gpu, m, n, 130, xt, wt, pads=(1, 1, 3), offset=1, added=True)


@pytest.mark.parametrize("xt,wt", ORDERS)
@pytest.mark.parametrize("m", [1, 20, 33, 64, 100, 300])
def test_logits_of_a_text_head(gpu, m, xt, wt):
    product(gpu, m, 151936, 72, xt, wt)
    if m in (1, 64):
        product(gpu, m, 151936, 201, xt, wt, pads=(1, 1, 0), offset=1, added=True)


def test_more_outputs_than_a_launch_of_few_rows(gpu):
    """16 outputs a workgroup, 2^20 workgroups a launch: the second launch's outputs"""
    product(gpu, 1, (1 << 24) + 21, 8)


@pytest.mark.parametrize("xt", [False, True])
def test_more_tiles_than_a_launch(gpu, xt):
    """128 rows a tile, 2^22 tiles a launch: the second launch's rows"""
    import hiprt
    m = (1 << 29) + 300
    i = np.random.default_rng(17).integers(0, 5, m, np.uint8)
    with R.Arena() as D:
        y = D.room(4 * m, 0xee)
        assert gpu.dense_raw(D.put(BITS[i]).ptr, m if xt else 1, D.put(BITS[4:]).ptr, 1, m, 1, 1, y.ptr, 1, gpu.DTYPE_F32,
                             x_transposed=xt) == 0
        hiprt.synchronize()
        assert np.array_equal(y.download((m,), np.float32), (2 * VALUES)[i])


def test_more_columns_than_a_launch_of_sums(gpu):
    """the bias gradient of 2^26 columns and 37: 16 a workgroup, 2^22 workgroups a launch"""
    import hiprt
    m, n = 2, (1 << 26) + 37
    rng = np.random.default_rng(14)
    bits, v = whole_numbers(rng, m, n)
    with R.Arena() as D:
        dbias = D.room(4 * n, 0xee)
        assert gpu.dense_activation_backward_raw(D.put(bits).ptr, n, None, 0, m, n, 0, None, 0, dbias.ptr) == 0
        hiprt.synchronize()
        assert np.array_equal(dbias.download((n,), np.float32), v[0] + v[1])
        assert gpu.lib().d3s_stream_workspace_release(None) == 0


def test_one_row_in_place_has_no_stride(gpu):
    """one row's strides say nothing: any pair is taken in place"""
    import hiprt
    rng = np.random.default_rng(15)
    n, k = 40, 24
    (xb, x), (wb, w), (gb, g) = whole_numbers(rng, 1, k), whole_numbers(rng, n, k), whole_numbers(rng, 1, n)
    r = rng.integers(-100, 100, n).astype(np.float32)
    with R.Arena() as D:
        y, dy = D.put(r), D.put(gb)
        assert gpu.dense_raw(D.put(xb).ptr, k, D.put(wb).ptr, k, 1, n, k, y.ptr, n, gpu.DTYPE_F32, residual=y.ptr,
                             residual_stride=n + 9) == 0
        assert gpu.dense_activation_backward_raw(dy.ptr, n + 5, None, 0, 1, n, 0, dy.ptr, n, None) == 0
        hiprt.synchronize()
        assert np.array_equal(y.download((n,), np.float32), r + (x @ w.T)[0])
        assert np.array_equal(dy.download((n,), np.uint16), gb[0])


@pytest.mark.parametrize("n", [1, 5, 7, 8, 9])
def test_very_few_outputs_by_the_inner_index(gpu, n):
    """so many rows that large tiles pay, outputs fewer than what those turn at a time"""
    product(gpu, 57344, n, 1024, False, True)
    product(gpu, 50000, n, 1090, False, True, added=True)


def test_the_time_of_very_few_outputs(gpu):
    """five outputs by the inner index take no longer than eight, a few per cent aside (they took 3.3 times
    as long in tiles whose loads are made for eight)"""
    import ctypes

    import hiprt
    m, k = 57344, 8192
    H = hiprt.hip()
    start, stop = ctypes.c_void_p(), ctypes.c_void_p()
    hiprt.check(H.hipEventCreate(ctypes.byref(start)))
    hiprt.check(H.hipEventCreate(ctypes.byref(stop)))
    times = {}
    with R.Arena() as D:
        x, w, y = D.room(2 * m * k, 0), D.room(2 * 8 * k, 0), D.room(4 * 8 * m)
        for n in (5, 8):
            for _ in range(4):
                hiprt.check(H.hipEventRecord(start, None))
                assert gpu.dense_raw(x.ptr, k, w.ptr, n, m, n, k, y.ptr, n, gpu.DTYPE_F32, w_transposed=True) == 0
                hiprt.check(H.hipEventRecord(stop, None))
                hiprt.synchronize()
                ms = ctypes.c_float()
                hiprt.check(H.hipEventElapsedTime(ctypes.byref(ms), start, stop))
                times[n] = min(times.get(n, 1e9), ms.value)
    H.hipEventDestroy(start)
    H.hipEventDestroy(stop)
    assert times[5] < 1.7 * times[8], times
