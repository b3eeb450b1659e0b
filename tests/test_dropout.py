"""Dropout against a plain form in 64 bits: the mask is the generator's, place by place."""
import numpy as np
import pytest

import step_ref as SR
import train_ref as R

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 1}
SIZE = {"f32": 4, "bf16": 2}
SEED, DRAW = 0x123456789ABCDEF0, (7 << 32) | 5


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


def run(gpu, x, residual, dtype, p, seed=SEED, draw=DRAW, add=None, strides=None, lead=0, inplace=None, stream=None):
    """x, residual bits [n, W]; strides: x's, residual's and y's paddings"""
    import hiprt
    n, width = x.shape
    px, pr, py = strides or (0, 0, 0)
    es = SIZE[dtype]
    with R.Arena() as D:
        bx = D.put(R.with_stride(x, width + px, lead))
        br = None if residual is None else D.put(R.with_stride(residual, width + pr, lead))
        by = {"x": bx, "residual": br}[inplace] if inplace else D.room(es * (n * (width + py) + lead), 0xee)
        ba = D.put(np.array([add], np.uint64)) if add is not None else None
        rc = gpu.dropout_raw(bx.ptr + lead * es, CODE[dtype], width + px, br.ptr + lead * es if br else None, width + pr, n, width,
                             p, seed, draw, ba.ptr if ba else None, by.ptr + lead * es, width + py, stream=stream)
        assert rc == 0
        hiprt.synchronize()
        flat = by.download((lead + n * (width + py) - py,), np.uint16 if dtype == "bf16" else np.float32)
        if not inplace:
            gaps = np.concatenate([flat[lead + r * (width + py) + width: lead + (r + 1) * (width + py)] for r in range(n - 1)] or [flat[:0]])
            assert (np.ascontiguousarray(gaps).view(np.uint8) == 0xee).all()
        return R.rows_at(flat, n, width, width + py, lead)


def check(got, x, residual, dtype, p, seed=SEED, draw=DRAW):
    ref, kept = SR.dropout(x, p, seed, draw, residual)
    # the scale's rounding, the product's and the sum's, then the output's
    part = np.abs(ref if residual is None else ref - residual)
    R.assert_near(R.from_bits(got), ref, SR.U * (2 * part + np.abs(ref)) + SR.half_step(dtype) * np.abs(ref) * 1.01 + 1e-38)
    return kept


SHAPES = [(1, 1), (1, 7), (3, 64), (5, 100), (7, 101), (2, 2048), (300, 33), (4, 4097), (9, 515), (1000, 8), (1, 100003), (33, 2050)]


@pytest.mark.parametrize("n,width", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("strides,lead", [((0, 0, 0), 0), ((3, 0, 8), 1)])
def test_dropout(gpu, n, width, dtype, strides, lead):
    rng = np.random.default_rng([n, width])
    (xb, x), (rb, r) = (R.to_bits(rng.standard_normal((n, width)), dtype) for _ in range(2))
    for p, res in ((0.1, True), (0.5, False), (0.9, True)):
        kept = check(run(gpu, xb, rb if res else None, dtype, p, strides=strides, lead=lead), x, r if res else None, dtype, p)
        if n * width > 1000:  # five deviations
            assert abs(kept.mean() - (1 - p)) < 5 * np.sqrt(p * (1 - p) / kept.size)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -24, 2.0 ** -25, 1 - 2.0 ** -24, 1.0])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_ends_of_p(gpu, p, dtype):
    xb, x = R.to_bits(np.random.default_rng(1).standard_normal((20, 333)), dtype)
    got = run(gpu, xb, None, dtype, p)
    kept = check(got, x, None, dtype, p)
    if p == 0:
        assert np.array_equal(got.view(np.uint8), xb.view(np.uint8))
    if p == 1:
        assert not kept.any() and (got == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_gradient_is_the_same_call(gpu, dtype):
    """where y = x / (1 - p) the gradient passes, elsewhere it is 0: differences of a linear map"""
    rng = np.random.default_rng(2)
    (xb, x), (db, dy) = (R.to_bits(rng.standard_normal((11, 203)), dtype) for _ in range(2))
    y, dx = run(gpu, xb, None, dtype, 0.4), run(gpu, db, None, dtype, 0.4, strides=(5, 0, 1))
    assert np.array_equal(R.from_bits(y) == 0, R.from_bits(dx) == 0)
    check(dx, dy, None, dtype, 0.4)


def test_the_mask_is_uniform_fills(gpu):
    u = gpu.uniform_fill(7 * 131, 99, 12).reshape(7, 131)
    x = np.ones((7, 131), np.float32)
    assert np.array_equal(run(gpu, x, None, "f32", 0.3, seed=99, draw=12) > 0, u >= np.float32(0.3))


def test_other_seeds_draws_and_the_device_counter(gpu):
    x = np.ones((40, 50), np.float32)
    a = run(gpu, x, None, "f32", 0.5)
    for kw in (dict(seed=SEED + 1), dict(seed=SEED ^ (1 << 63)), dict(draw=DRAW + 1), dict(draw=DRAW ^ (1 << 40))):
        assert not np.array_equal(run(gpu, x, None, "f32", 0.5, **kw), a)
    assert np.array_equal(run(gpu, x, None, "f32", 0.5, draw=DRAW - 3, add=3), a)
    assert np.array_equal(run(gpu, x, None, "f32", 0.5, draw=(1 << 64) - 2, add=DRAW + 2), a)


@pytest.mark.parametrize("n,width,pad", [(5, 101, 0), (6, 64, 0), (4, 37, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_in_place(gpu, n, width, pad, dtype):
    rng = np.random.default_rng(3)
    x, r = (R.to_bits(rng.standard_normal((n, width)), dtype)[0] for _ in range(2))
    apart = run(gpu, x, r, dtype, 0.25)
    for where in ("x", "residual"):
        got = run(gpu, x, r, dtype, 0.25, strides=(pad, pad, pad), inplace=where)
        assert np.array_equal(got.view(np.uint8), apart.view(np.uint8))


def test_dropped_infinities_and_nan_are_zeros(gpu):
    x = np.full((10, 77), np.nan, np.float32)
    x[::2] = np.inf
    got = run(gpu, x, None, "f32", 0.5)
    kept = SR.uniforms(x.size, SEED, DRAW).reshape(x.shape) >= 0.5
    assert (got[~kept] == 0).all() and np.isnan(got[1::2][kept[1::2]]).all() and np.isposinf(got[::2][kept[::2]]).all()


def test_counters_past_32_bits(gpu):
    """rows whose elements' numbers pass 2^32: a row's mask by its own numbers"""
    n, width = 3, 1 << 31
    import hiprt
    if hiprt.free_memory() < 40 << 30:
        pytest.skip("not enough memory")
    with R.Arena() as D:
        b = D.room(2 * n * (width - 1), 0x3f)  # bf16 0.747
        assert gpu.dropout_raw(b.ptr, 1, width - 1, None, 0, n, width - 1, 0.5, SEED, DRAW, None, b.ptr, width - 1) == 0
        hiprt.synchronize()
        first = 2 * (width - 1) + 1000  # in the last row, past 2^32
        got = b.download((4096,), np.uint16, offset=2 * first)
    q = np.arange(first // 4, (first + 4096) // 4 + 1, dtype=np.uint64)
    import d3s_workloads as W
    words = W.philox4x32_10([(q & np.uint64(0xffffffff)).astype(np.uint32), (q >> np.uint64(32)).astype(np.uint32),
                             np.full(len(q), DRAW & 0xffffffff, np.uint32), np.full(len(q), DRAW >> 32, np.uint32)],
                            SEED & 0xffffffff, SEED >> 32)
    w = np.stack(words, 1).reshape(-1)[first % 4:first % 4 + 4096]
    assert first + 4096 > 1 << 32
    assert np.array_equal(got != 0, (w >> np.uint32(31)) == 1)
