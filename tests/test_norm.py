"""Root-mean-square norm with the residual's addition, its 8-bit output and its gradient
against a plain form in 64 bits."""
import numpy as np
import pytest

import step_ref as SR
import train_ref as R

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 1, "e4m3": 2}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}
NP = {"f32": np.float32, "bf16": np.uint16, "e4m3": np.uint8}


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


def forward(gpu, x, residual, gain, eps, dtype, out, group=0, pad=0, lead=0, keep=True, inplace=None, stream=None):
    """x, residual bits [n, W]; dict of sum (bits), y (bits), rstd, scales.  inplace: "sum=residual",
    "sum=x", "y=x" or "y=residual" """
    import hiprt
    n, width = x.shape
    S, es = width + pad, SIZE[dtype]
    with R.Arena() as D:
        put = lambda b: D.put(R.with_stride(b, S, lead))  # noqa: E731
        bx, br = put(x), None if residual is None else put(residual)
        at = lambda b, size=es: None if b is None else b.ptr + lead * size  # noqa: E731
        bsum = D.room(es * (n * S + lead), 0xee) if keep else None
        by = D.room(SIZE[out] * (n * S + lead), 0xee)
        where = {"sum=residual": ("s", br), "sum=x": ("s", bx), "y=x": ("y", bx), "y=residual": ("y", br)}.get(inplace)
        if where:
            if where[0] == "s":
                bsum = where[1]
            else:
                by = where[1]
        groups = -(-width // (group or width))
        scales, rstd = D.room(4 * n * groups, 0xee), D.room(4 * n, 0xee)
        rc = gpu.rms_norm_raw(at(bx), CODE[dtype], S, at(br), S, at(bsum), S, D.put(gain).ptr if gain is not None else None, eps,
                              n, width, at(by, SIZE[out]), CODE[out], S, group=group, scales=scales.ptr, rstd=rstd.ptr, stream=stream)
        assert rc == 0
        hiprt.synchronize()

        def rows(b, t):
            flat = b.download((lead + n * S - pad,), NP[t])
            if not where:
                gaps = np.concatenate([flat[lead + r * S + width: lead + (r + 1) * S] for r in range(n - 1)] or [flat[:0]])
                assert (np.ascontiguousarray(gaps).view(np.uint8) == 0xee).all(), "written between two rows"
            return R.rows_at(flat, n, width, S, lead)

        return dict(sum=rows(bsum, dtype) if bsum else None, y=rows(by, out), rstd=rstd.download((n,), np.float32),
                    scales=scales.download((n, groups), np.float32))


WIDTHS = [(1, 2048), (3, 1), (5, 7), (300, 64), (33, 100), (70, 128), (9, 513), (4, 1000), (2, 2050), (7, 4096), (3, 5001),
          (2, 8192), (2, 16384), (3, 16391), (1, 70001), (2000, 40), (1100, 2048)]


@pytest.mark.parametrize("n,width", WIDTHS)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_norm(gpu, n, width, dtype, out):
    rng = np.random.default_rng([n, width])
    (xb, x), (rb, r) = (R.to_bits(rng.standard_normal((n, width)) * s, dtype) for s in (1.0, 3.0))
    gb, g = R.to_bits(1 + 0.3 * rng.standard_normal(width), dtype)
    pad, lead = (0, 0) if width % 2 == 0 else (3, 1)
    for res, keep in ((None, False), (r, True)):
        got = forward(gpu, xb, None if res is None else rb, gb if keep else None, 1e-5, dtype, out, pad=pad, lead=lead, keep=keep)
        h = x if res is None else x + r
        y, rstd = SR.norm(h, g if keep else np.ones(width), float(np.float32(1e-5)))
        steps = SR.norm_steps(width)
        R.assert_near(got["rstd"], rstd, SR.U * steps * rstd, "rstd")
        R.assert_near(R.from_bits(got["y"]), y, SR.U * (steps + 4) * np.abs(y) + SR.half_step(out) * np.abs(y) * 1.01 + 1e-38, "y")
        if keep:
            R.assert_near(R.from_bits(got["sum"]), h, (SR.half_step(dtype) * 1.01 + SR.U) * np.abs(h), "sum")


@pytest.mark.parametrize("n,width", [(1, 2048), (5, 7), (40, 64), (33, 100), (9, 513), (3, 2050), (2, 8192), (3, 16391), (600, 256), (1100, 2048)])
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
def test_8_bits(gpu, n, width, group):
    rng = np.random.default_rng([n, width, group])
    dtype = "bf16" if group != 64 else "f32"
    (xb, x), (rb, r) = (R.to_bits(rng.standard_normal((n, width)) * np.exp(2 * rng.standard_normal((n, 1))), dtype) for _ in range(2))
    gb, g = R.to_bits(1 + 0.3 * rng.standard_normal(width), dtype)
    pad = 0 if width % 2 == 0 else 5
    got = forward(gpu, xb, rb, gb, 1e-6, dtype, "e4m3", group=group, pad=pad)
    y, _ = SR.norm(x + r, g, float(np.float32(1e-6)))
    size = group or width
    groups = -(-width // size)
    most = np.stack([np.abs(y[:, c * size:(c + 1) * size]).max(1) for c in range(groups)], 1)
    steps = SR.norm_steps(width) + 6
    R.assert_near(got["scales"], most / 448, SR.U * steps * most / 448, "scales")
    scale = np.repeat(got["scales"].astype(np.float64), size, 1)[:, :width]
    stands = SR.e4m3_values()[got["y"]] * scale
    # half a step of 2^-3 of the value's power of two, or of the smallest, 2^-9
    R.assert_near(stands, y, np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * scale) * (1 + 1e-5) + SR.U * steps * np.abs(y), "q")
    # the greatest of each group is 448 (its quotient by the scale, which is rounded, still rounds there)
    q = np.abs(SR.e4m3_values()[got["y"]])
    assert all((q[:, c * size:(c + 1) * size].max(1) == 448).all() for c in range(groups))


@pytest.mark.parametrize("width", [40, 513, 2048, 16391])
def test_zeros_infinities_and_nan(gpu, width):
    n = 6
    rng = np.random.default_rng(width)
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[0] = 0
    x[1, width // 2] = np.inf
    x[2, width - 1] = np.nan
    x[3, :32] = 0
    x[4] *= np.float32(1e-25)  # squares below the least subnormal
    got = forward(gpu, x, None, None, 1e-6, "f32", "f32")
    h = x.astype(np.float64)
    sq = (x * x).astype(np.float64)  # (the squares in 32 bits)
    assert (got["y"][0] == 0).all() and np.isnan(got["y"][1, width // 2]) and got["rstd"][1] == 0
    assert (got["y"][1, np.arange(width) != width // 2] == 0).all()
    assert np.isnan(got["y"][2]).all() and np.isnan(got["rstd"][2])
    ref = h / np.sqrt(sq.mean(1, keepdims=True) + float(np.float32(1e-6)))
    for row in (3, 4, 5):
        R.assert_near(got["y"][row], ref[row], SR.U * (SR.norm_steps(width) + 4) * np.abs(ref[row]) + 1e-38)
    for group in (0, 32):
        q = forward(gpu, x, None, None, 1e-6, "f32", "e4m3", group=group)
        v = SR.e4m3_values()[q["y"]]
        assert (q["scales"][0] == 0).all() and (v[0] == 0).all()
        assert np.isnan(q["scales"][2]).all() and np.isnan(v[2]).all()
        size = group or width
        where = (width // 2) // size
        assert np.isnan(q["scales"][1, where]) and np.isnan(v[1, where * size:(where + 1) * size]).all()
        assert (q["scales"][1, np.arange(q["scales"].shape[1]) != where] == 0).all()
        if group:
            assert q["scales"][3, 0] == 0 and (v[3, :32] == 0).all()


@pytest.mark.parametrize("width", [64, 100, 2048, 5000, 20000])
@pytest.mark.parametrize("inplace", ["sum=residual", "sum=x", "y=x", "y=residual"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_in_place(gpu, width, inplace, dtype):
    rng = np.random.default_rng(width)
    n = 5
    x, r = (R.to_bits(rng.standard_normal((n, width)), dtype)[0] for _ in range(2))
    keep = inplace.startswith("sum")
    apart = forward(gpu, x, r, None, 1e-6, dtype, dtype, keep=keep)
    got = forward(gpu, x, r, None, 1e-6, dtype, dtype, keep=keep, inplace=inplace)
    for name in ("y", "rstd") + (("sum",) if keep else ()):
        assert np.array_equal(got[name].view(np.uint8), apart[name].view(np.uint8)), name


def backward(gpu, dy, h, gain, rstd, dsum, dtype, pad=0, lead=0, dgain=True, dx=True, inplace=None, stream=None, workspace=None):
    import hiprt
    n, width = dy.shape
    S, es = width + pad, SIZE[dtype]
    with R.Arena() as D:
        put = lambda b: D.put(R.with_stride(b, S, lead))  # noqa: E731
        at = lambda b: None if b is None else b.ptr + lead * es  # noqa: E731
        bd, bh, bs = put(dy), put(h), None if dsum is None else put(dsum)
        bx = {"dy": bd, "h": bh, "dsum": bs}[inplace] if inplace else D.room(es * (n * S + lead), 0xee) if dx else None
        bg = D.room(4 * width, 0xee) if dgain else None
        if workspace == "own":
            W = gpu.Workspace(gpu.lib().d3s_rms_norm_backward_workspace_bytes(n, width, int(dgain)))
            D.held.append(W.buf)
            workspace = W.arg()
        rc = gpu.rms_norm_backward_raw(at(bd), CODE[dtype], S, at(bh), S, D.put(gain).ptr if gain is not None else None,
                                       D.put(np.asarray(rstd, np.float32)).ptr, at(bs), S, n, width, at(bx), S,
                                       bg.ptr if bg else None, stream=stream, workspace=workspace)
        assert rc == 0
        hiprt.synchronize()
        out = [None, bg.download((width,), np.float32) if bg else None]
        if bx:
            out[0] = R.rows_at(bx.download((lead + n * S - pad,), NP[dtype]), n, width, S, lead)
        return out


@pytest.mark.parametrize("n,width", WIDTHS + [(5000, 16), (700, 513), (257, 8192)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradient(gpu, n, width, dtype):
    rng = np.random.default_rng([n, width, 5])
    (db, dy), (hb, h), (sb, dsum) = (R.to_bits(rng.standard_normal((n, width)), dtype) for _ in range(3))
    gb, g = R.to_bits(1 + 0.3 * rng.standard_normal(width), dtype)
    rstd = (1 / np.sqrt((h * h).mean(1) + 1e-6)).astype(np.float32)
    pad, lead = (0, 0) if width % 2 == 0 else (3, 1)
    for gain, res in ((True, True), (False, False)):
        got, dgain = backward(gpu, db, hb, gb if gain else None, rstd, sb if res else None, dtype, pad, lead)
        ref, err, ref_g, size = SR.norm_grad(dy, h, g if gain else np.ones(width), rstd.astype(np.float64), dsum if res else None)
        R.assert_near(R.from_bits(got), ref, err + SR.half_step(dtype) * np.abs(ref) * 1.01, "dx")
        R.assert_near(dgain, ref_g, SR.U * (n + 4) * size, "dgain")
    # the same bits with a workspace of the caller's, for either output alone, and in place
    got, dgain = backward(gpu, db, hb, gb, rstd, sb, dtype, pad, lead)
    again = backward(gpu, db, hb, gb, rstd, sb, dtype, pad, lead, workspace="own")
    assert np.array_equal(again[0].view(np.uint8), got.view(np.uint8)) and np.array_equal(again[1].view(np.uint32), dgain.view(np.uint32))
    assert np.array_equal(backward(gpu, db, hb, gb, rstd, sb, dtype, pad, lead, dgain=False)[0].view(np.uint8), got.view(np.uint8))
    assert np.array_equal(backward(gpu, db, hb, gb, rstd, sb, dtype, pad, lead, dx=False)[1].view(np.uint32), dgain.view(np.uint32))
    for where in ("dy", "h", "dsum"):
        same = backward(gpu, db, hb, gb, rstd, sb, dtype, pad, lead, inplace=where)
        assert np.array_equal(same[0].view(np.uint8), got.view(np.uint8)), where
        assert np.array_equal(same[1].view(np.uint32), dgain.view(np.uint32)), where


def test_gradient_is_the_norms(gpu):
    """central differences of the 64-bit norm"""
    rng = np.random.default_rng(8)
    n, width = 3, 11
    h, dy = rng.standard_normal((n, width)).astype(np.float32), rng.standard_normal((n, width)).astype(np.float32)
    g = (1 + 0.3 * rng.standard_normal(width)).astype(np.float32)
    eps = 1e-3
    _, rstd = SR.norm(h.astype(np.float64), g, eps)
    dx, dgain = backward(gpu, dy, h, g, rstd, None, "f32")
    f = lambda hh, gg: (SR.norm(hh, gg, eps)[0] * dy).sum()  # noqa: E731
    step = 1e-5
    for r in range(n):
        for j in range(width):
            e = np.zeros((n, width))
            e[r, j] = step
            d = (f(h + e, g) - f(h - e, g)) / (2 * step)
            assert abs(d - dx[r, j]) < 2e-5 * (1 + np.abs(dy).sum())
    for j in range(width):
        e = np.zeros(width)
        e[j] = step
        d = (f(h.astype(np.float64), g + e) - f(h.astype(np.float64), g - e)) / (2 * step)
        assert abs(d - dgain[j]) < 2e-5 * (1 + np.abs(dy).sum())


def test_no_rows(gpu):
    import hiprt
    with R.Arena() as D:
        g = D.room(4 * 30, 0xee)
        assert gpu.rms_norm_backward_raw(None, 1, 30, None, 30, None, None, None, 0, 0, 30, None, 0, g.ptr) == 0
        hiprt.synchronize()
        assert (g.download((30,), np.float32) == 0).all()


WIDER = [(3, 2051), (5, 2560), (2, 3333), (3, 4100), (2, 5120), (2, 6001), (2, 7168), (2, 8191), (2, 8194), (2, 10240), (2, 12000),
         (2, 14337), (600, 2600), (300, 9000)]


@pytest.mark.parametrize("n,width", WIDER)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_norm_of_wider_rows(gpu, n, width, dtype, out):
    """workgroups of every number of threads"""
    test_norm(gpu, n, width, dtype, out)


@pytest.mark.parametrize("n,width", WIDER)
@pytest.mark.parametrize("group", [0, 64, 256])
def test_8_bits_of_wider_rows(gpu, n, width, group):
    test_8_bits(gpu, n, width, group)


@pytest.mark.parametrize("n,width,group", [(1500, 2048, 128), (3000, 1000, 0), (2000, 40, 32), (150, 16391, 0), (150, 16391, 64), (600, 4100, 256)])
def test_8_bits_are_the_quotients(gpu, n, width, group):
    """every y is the fp32 quotient by its group's scale, rounded to the nearest even: equal, from the same rstd (the
    products are fp32's own, one after the other)"""
    rng = np.random.default_rng([n, width, group, 9])
    x = (rng.standard_normal((n, width)) * np.exp(rng.uniform(-3, 3, (n, 1)))).astype(np.float32)
    g = (1 + 0.3 * rng.standard_normal(width)).astype(np.float32)
    x[:2] *= np.array([[1e-33], [1e-41]], np.float32)  # scales below 2^-100, subnormal ones
    got = forward(gpu, x, None, g, 1e-6, "f32", "e4m3", group=group)
    y = x * got["rstd"][:, None] * g
    size = group or width
    most = np.stack([np.abs(y[:, c:c + size]).max(1) for c in range(0, width, size)], 1)
    assert np.array_equal(got["scales"], most / np.float32(448))
    q = y / np.repeat(got["scales"], size, 1)[:, :width]
    assert q.dtype == np.float32
    v = SR.e4m3_values()[:127]
    middle = (v[1:] + v[:-1]) / 2  # exact in fp32
    at = np.searchsorted(middle, np.abs(q).astype(np.float64))  # (a tie: the lower)
    tie = (at < 126) & (np.abs(q) == middle[np.minimum(at, 125)])
    at += tie & (at % 2 == 1)
    assert np.array_equal(got["y"], (at | np.where(np.signbit(q), 128, 0)).astype(np.uint8)), (got["y"] != (at | np.where(np.signbit(q), 128, 0))).sum()


@pytest.mark.parametrize("n,width", WIDTHS + [(5000, 16), (20001, 100), (700, 513), (257, 8192), (1025, 1025), (3000, 3000), (40, 20000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_column_sums_of_whole_numbers(gpu, n, width, dtype):
    """dgain of whole dy and h and of rstd that are powers of two: equal, so that no row is lost or taken twice"""
    rng = np.random.default_rng([n, width, 17])
    whole = lambda: R.to_bits(rng.integers(1, 9, (n, width)) * rng.choice([-1, 1], (n, width)), dtype)  # noqa: E731
    (db, dy), (hb, h) = whole(), whole()
    rstd = rng.choice([0.25, 0.5, 1.0], n).astype(np.float32)
    want = (dy * h * rstd[:, None]).sum(0)
    assert (np.abs(dy * h).sum(0) < 2 ** 22).all()
    for dx in (True, False):
        assert np.array_equal(backward(gpu, db, hb, None, rstd, None, dtype, dx=dx)[1], want)
