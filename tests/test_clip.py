"""The global norm of many gradients and clipping, against 64 bits: lengths from
none up, every alignment, both types, in place and not, norms that do not clip,
overflow in 32 bits or are not finite."""
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


def run(gpu, tensors, max_norm, in_place=False, norm_only=False, use_ws=False, shift=0):
    """tensors: list of (bits, offset in elements)"""
    import hiprt
    with R.Arena() as D:
        src, dst, bufs = [], [], []
        for bits, at in tensors:
            room = np.full(at + bits.size + 16, 0x1234, bits.dtype) if bits.dtype == np.uint16 else \
                np.full(at + bits.size + 16, 7.5, bits.dtype)
            held = room.copy()
            held[at:at + bits.size] = bits
            a = D.put(held)
            to = at if in_place else at + shift
            b = a if in_place else D.put(room)
            src.append(a.ptr + at * bits.itemsize)
            dst.append(b.ptr + to * bits.itemsize)
            bufs.append((b, to, held if in_place else room))
        src, dst = np.array(src, np.uint64), np.array(dst, np.uint64)
        numel = np.array([b.size for b, _ in tensors], np.int64)
        dt = np.array([1 if b.dtype == np.uint16 else 0 for b, _ in tensors], np.int32)
        norm = D.room(4, 0xee)
        ws = None
        if use_ws:
            W = gpu.Workspace(gpu.lib().d3s_clip_grads_workspace_bytes(len(tensors)))
            D.held.append(W.buf)
            ws = W.arg()
        rc = gpu.clip_grads_raw(src.ctypes.data, None if norm_only else dst.ctypes.data, numel.ctypes.data,
                                dt.ctypes.data, len(tensors), max_norm, norm.ptr, workspace=ws)
        assert rc == 0
        hiprt.synchronize()
        out = []
        for (b, at, room), (bits, _) in zip(bufs, tensors):
            flat = b.download(room.shape, bits.dtype)
            keep = np.ones(room.size, bool)
            keep[at:at + bits.size] = False
            assert np.array_equal(flat[keep], room[keep]), "written outside"
            out.append(flat[at:at + bits.size])
        return float(norm.download((1,), np.float32)[0]), out


def check(got_norm, got, tensors, max_norm):
    norm = math.sqrt(math.fsum(float((R.from_bits(b) ** 2).sum()) for b, _ in tensors))
    # the sums are exact to 2^-40 of the norm; one rounding to fp32
    assert abs(got_norm - norm) <= 1.01 * R.U * norm + 1e-45
    clipped = norm > max_norm
    for out, (b, _) in zip(got, tensors):
        ref = R.from_bits(b)
        if not clipped:
            assert np.array_equal(out.view(np.uint8), b.view(np.uint8))
            continue
        ref = ref * (max_norm / norm)
        # the norm, the quotient and the product round once each, then the result to its type (or below its range)
        tol = 4 * R.U * np.abs(ref) + (R.BF16 * np.abs(ref) + 2.0 ** -134 if b.dtype == np.uint16 else 2.0 ** -149)
        R.assert_near(R.from_bits(out), ref, tol)


def tensors_of(sizes, seed=0, scale=0.02):
    rng = np.random.default_rng([len(sizes), seed])
    out = []
    for i, n in enumerate(sizes):
        bits, _ = R.to_bits(rng.standard_normal(n) * scale, "bf16" if rng.random() < 0.5 else "f32")
        out.append((bits, int(rng.integers(0, 9))))
    return out


@pytest.mark.parametrize("sizes", [
    [1], [0, 0, 5, 0], [3, 1, 8, 7, 9, 16, 15, 17], [1023, 1024, 1025, 2047, 4096, 4097], [100003, 1, 2],
    [4097 * 2048, 2048, 0, 4096], [37] * 127, [37] * 128, [5, 0] * 200, list(range(300)), [2500000, 3]])
def test_clip(gpu, sizes):
    t = tensors_of(sizes)
    norm = math.sqrt(sum(float((R.from_bits(b) ** 2).sum()) for b, _ in t))
    for limit in (norm / 3, norm * 2):
        limit = float(np.float32(limit))
        check(*run(gpu, t, limit), t, limit)
        check(*run(gpu, t, limit, shift=3, use_ws=True), t, limit)
        check(*run(gpu, t, limit, in_place=True), t, limit)
    n, out = run(gpu, t, 1.0, norm_only=True)
    check(n, [], t, 1.0)


def test_nothing(gpu):
    assert run(gpu, [], 1.0)[0] == 0.0
    t = [(np.zeros(0, np.float32), 0)] * 3
    assert run(gpu, t, 1.0)[0] == 0.0 and run(gpu, t, 1.0, norm_only=True)[0] == 0.0
    z = [(np.zeros(1000, np.float32), 1)]
    assert run(gpu, z, 1.0)[0] == 0.0


def test_squares_past_fp32(gpu):
    """squares that overflow or vanish in 32 bits do neither here"""
    for scale in (1e25, 1e-30):
        b = np.float32(np.random.default_rng(1).standard_normal(5000) * scale)
        t = [(b, 1), (R.to_bits(b[:777], "bf16")[0], 0)]
        norm = math.sqrt(sum(float((R.from_bits(x) ** 2).sum()) for x, _ in t))
        limit = float(np.float32(norm / 7))
        check(*run(gpu, t, limit), t, limit)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("in_place", [False, True])
def test_not_finite(gpu, bad, in_place):
    t = tensors_of([100, 5000], 3)
    b = np.float32(np.linspace(-1, 1, 300))
    b[200] = bad
    t.append((b, 2))
    n, out = run(gpu, t, 0.5, in_place=in_place)
    assert not math.isfinite(n)
    for o, (x, _) in zip(out, t):
        assert np.array_equal(o.view(np.uint8), x.view(np.uint8))


def test_one_tensor_past_32_bits(gpu):
    """2^32 + 11 elements, in place"""
    import hiprt
    n = (1 << 32) + 11
    with R.Arena() as D:
        big = D.room(2 * n, 0x3c)  # every element 0x3c3c
        v = float(R.from_bits(np.array([0x3c3c], np.uint16))[0])
        src, numel, dt = np.array([big.ptr], np.uint64), np.array([n], np.int64), np.array([1], np.int32)
        out = D.room(4)
        assert gpu.clip_grads_raw(src.ctypes.data, src.ctypes.data, numel.ctypes.data, dt.ctypes.data, 1, 100.0, out.ptr) == 0
        hiprt.synchronize()
        norm = v * math.sqrt(n)
        assert abs(float(out.download((1,), np.float32)[0]) - norm) <= 1.01 * R.U * norm
        want = R.to_bits(np.array([v * (100.0 / norm)]), "bf16")[0][0]
        for at in (0, 1 << 20, (1 << 31) - 5, (1 << 32) - 7, n - 11):
            assert (big.download((11,), np.uint16, 2 * at) == want).all()


def test_the_same_bits_each_time(gpu):
    t = tensors_of([50000, 3, 777, 120000], 5)
    a = run(gpu, t, 0.5)
    for _ in range(3):
        b = run(gpu, t, 0.5)
        assert a[0] == b[0] and all(np.array_equal(x, y) for x, y in zip(a[1], b[1]))
