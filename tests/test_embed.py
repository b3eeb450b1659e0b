"""Embedding lookup and its gradient against a plain form in 64 bits."""
import numpy as np
import pytest

import step_ref as SR
import train_ref as R

pytestmark = pytest.mark.gpu
CODE = {"f32": 0, "bf16": 1}
SIZE = {"f32": 4, "bf16": 2}


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


def make_ids(rng, n, t, vocab, how):
    if how == "same":
        ids = np.full((n, t), vocab // 2)
    elif how == "zipf":
        ids = np.minimum(np.exp(rng.random((n, t)) * np.log(vocab + 1)) - 1, vocab - 1).astype(np.int64)
    else:
        ids = rng.integers(0, vocab, (n, t))
    odd = rng.random((n, t))
    ids = np.where(odd < 0.05, -1, np.where(odd > 0.97, vocab, ids))
    ids = np.where((odd > 0.5) & (odd < 0.52), 2 ** 31 - 1, ids)
    return ids.astype(np.int32)


@pytest.mark.parametrize("n,t,vocab,slot_rows,width,dtype,out,pad,lead", [
    (1, 10, 97, 97, 2048, "bf16", "bf16", 0, 0), (5, 1, 1000, 0, 1, "f32", "f32", 0, 0), (33, 3, 50, 0, 129, "bf16", "f32", 3, 1),
    (17, 64, 5, 5, 40, "f32", "bf16", 1, 3), (700, 2, 300, 311, 8, "bf16", "bf16", 0, 0), (4, 1, 7, 9, 5001, "bf16", "bf16", 0, 0),
    (3000, 1, 2000, 0, 64, "f32", "f32", 4, 0), (2, 11, 40, 0, 2049, "bf16", "f32", 0, 0)])
def test_lookup(gpu, n, t, vocab, slot_rows, width, dtype, out, pad, lead):
    import hiprt
    rng = np.random.default_rng([n, t, vocab, width])
    ids = make_ids(rng, n, t, vocab, "even")
    bits, table = R.to_bits(rng.standard_normal((SR.table_rows(t, vocab, slot_rows), width)), dtype)
    scale = np.float32(1.75)
    with R.Arena() as D:
        tab, y = D.put(R.with_stride(bits, width + pad, lead)), D.room(SIZE[out] * n * (width + pad), 0xee)
        rc = gpu.embed_raw(D.put(ids).ptr, n, t, tab.ptr + lead * SIZE[dtype], CODE[dtype], width + pad, vocab, slot_rows, width,
                           float(scale), y.ptr, CODE[out], width + pad)
        assert rc == 0
        hiprt.synchronize()
        flat = y.download((n * (width + pad),), np.uint16 if out == "bf16" else np.float32)
    got = R.from_bits(flat).reshape(n, width + pad)
    ref, size = SR.embed(ids, table, vocab, slot_rows, float(scale))
    R.assert_near(got[:, :width], ref, SR.U * (t + 1) * size + SR.half_step(out) * np.abs(ref) * 1.01)
    assert (flat.reshape(n, -1)[:, width:].view(np.uint8) == 0xee).all()


def grad(gpu, ids, bits, dtype, vocab, slot_rows, width, scale, out, dy_pad=0, pad=0, old=None, lead=0, stream=None,
         workspace=None):
    """the gradient's values (rows `pad` elements apart), and what lies between them"""
    import hiprt
    n, t = ids.shape
    rows = SR.table_rows(t, vocab, slot_rows)
    with R.Arena() as D:
        d = D.put(R.with_stride(bits, width + dy_pad, lead)) if n else D.room(16)
        g = D.room(SIZE[out] * rows * (width + pad), 0xee)
        if old is not None:
            g.upload(R.with_stride(old, width + pad))
        if workspace == "own":
            W = gpu.Workspace(gpu.lib().d3s_embed_backward_workspace_bytes(n, t, vocab, slot_rows, width))
            D.held.append(W.buf)
            workspace = W.arg()
        rc = gpu.embed_backward_raw(D.put(ids).ptr if ids.size else None, n, t, d.ptr + lead * SIZE[dtype], CODE[dtype],
                                    width + dy_pad, vocab, slot_rows, width, float(scale), old is not None, g.ptr, CODE[out],
                                    width + pad, stream=stream, workspace=workspace)
        assert rc == 0
        hiprt.synchronize()
        flat = g.download((rows, width + pad), np.uint16 if out == "bf16" else np.float32)
    if old is None:  # (the last row's padding may be the allocation's end)
        assert (np.ascontiguousarray(flat[:, width:]).view(np.uint8) == 0xee).all()
    return flat[:, :width]


GRADS = [
    # n, t, vocab, slot_rows, width, dtype, out, how, dy_pad, pad
    (1, 10, 97, 97, 64, "bf16", "f32", "even", 0, 0), (1, 1, 1, 0, 1, "f32", "f32", "even", 0, 0),
    (40, 1, 1000, 0, 130, "bf16", "bf16", "even", 3, 0), (300, 4, 50, 0, 72, "f32", "f32", "even", 0, 1),
    (1000, 1, 7, 0, 40, "bf16", "f32", "even", 0, 0), (513, 3, 60, 67, 2050, "bf16", "f32", "zipf", 1, 5),
    (2000, 1, 5000, 0, 16, "f32", "bf16", "zipf", 0, 0), (1500, 2, 100, 100, 24, "bf16", "f32", "same", 0, 0),
    (5000, 1, 30, 0, 8, "bf16", "bf16", "same", 0, 0), (9000, 1, 20011, 0, 33, "bf16", "f32", "zipf", 0, 0),
    (300, 1, 70000, 0, 9, "bf16", "f32", "even", 0, 0), (20000, 3, 513, 600, 8, "f32", "f32", "zipf", 0, 0),
    (70000, 1, 300000, 0, 8, "bf16", "f32", "zipf", 0, 0), (66000, 1, 50, 0, 12, "bf16", "f32", "zipf", 0, 0),
    (7001, 10, 333, 350, 16, "f32", "bf16", "zipf", 1, 0), (70003, 1, 3, 0, 5, "bf16", "f32", "same", 0, 0),
    (140001, 1, 1000000, 0, 4, "f32", "f32", "even", 0, 0), (33333, 3, 4097, 0, 40, "bf16", "f32", "zipf", 0, 0),
    (300000, 1, 8000, 0, 8, "bf16", "f32", "even", 0, 0), (40000, 1, 1000, 0, 17, "bf16", "bf16", "zipf", 0, 3),
    (16384, 2, 4096, 0, 12, "f32", "bf16", "zipf", 1, 0), (16383, 2, 4096, 0, 12, "f32", "f32", "zipf", 0, 0),
    (100000, 1, 1000, 0, 264, "bf16", "f32", "even", 0, 0),
    (1100, 64, 2000, 2048, 8, "bf16", "f32", "even", 0, 0), (3000, 1, 9, 0, 3000, "bf16", "bf16", "same", 0, 0), (64, 64, 33, 40, 56, "bf16", "bf16", "zipf", 0, 0)]


@pytest.mark.parametrize("n,t,vocab,slot_rows,width,dtype,out,how,dy_pad,pad", GRADS)
def test_gradient(gpu, n, t, vocab, slot_rows, width, dtype, out, how, dy_pad, pad):
    rng = np.random.default_rng([n, t, vocab, width])
    ids = make_ids(rng, n, t, vocab, how)
    bits, dy = R.to_bits(rng.standard_normal((n, width)), dtype)
    scale = np.float32(0.3)
    ref, size, count = SR.embed_grad(ids, dy, vocab, slot_rows, float(scale))
    # fp32 sums of `count` terms in any order, the scale, the rounding
    tol = SR.U * (count[:, None] + 2) * size + SR.half_step(out) * np.abs(ref) * 1.01
    lead = 1 if n % 2 else 0
    got = grad(gpu, ids, bits, dtype, vocab, slot_rows, width, scale, out, dy_pad, pad, lead=lead)
    R.assert_near(R.from_bits(got), ref, tol)
    assert (R.from_bits(got)[count == 0] == 0).all()
    again = grad(gpu, ids, bits, dtype, vocab, slot_rows, width, scale, out, dy_pad, pad, lead=lead, workspace="own")
    assert np.array_equal(again.view(np.uint8), got.view(np.uint8)), "another call, other bits"
    # added to what is there: rows that no id names keep their bits
    old, old_v = R.to_bits(rng.standard_normal(ref.shape), out)
    sums = grad(gpu, ids, bits, dtype, vocab, slot_rows, width, scale, out, dy_pad, pad, old=old, lead=lead)
    total = old_v + ref
    R.assert_near(R.from_bits(sums), total,
                  SR.U * ((count[:, None] + 2) * size + np.abs(total)) + SR.half_step(out) * np.abs(total) * 1.01)
    none = count == 0
    assert np.array_equal(np.ascontiguousarray(sums[none]), old[none])


def test_gradient_is_the_lookups(gpu):
    """differences: y is linear in the table, so <dy, y(table + e)> - <dy, y(table)> = e grad"""
    rng = np.random.default_rng(3)
    n, t, vocab, width = 12, 3, 6, 5
    ids = make_ids(rng, n, t, vocab, "even")
    bits, dy = R.to_bits(rng.standard_normal((n, width)), "f32")
    got = R.from_bits(grad(gpu, ids, bits, "f32", vocab, vocab, width, 1.5, "f32"))
    table = rng.standard_normal((t * vocab, width))
    base = (SR.embed(ids, table, vocab, vocab, 1.5)[0] * dy).sum()
    for r in range(t * vocab):
        for j in range(width):
            up = table.copy()
            up[r, j] += 1.0
            d = (SR.embed(ids, up, vocab, vocab, 1.5)[0] * dy).sum() - base
            assert abs(d - got[r, j]) < 1e-5 * (1 + np.abs(dy).sum())


def test_no_rows(gpu):
    ids = np.zeros((0, 3), np.int32)
    got = grad(gpu, ids, np.zeros((0, 16), np.float32), "f32", 50, 50, 16, 1.0, "f32")
    assert (got == 0).all()


def test_infinities_and_nan_stay_in_their_rows(gpu):
    rng = np.random.default_rng(4)
    n, vocab, width = 600, 90, 40
    ids = rng.integers(0, vocab, (n, 1)).astype(np.int32)
    bits, dy = R.to_bits(rng.standard_normal((n, width)), "f32")
    bits[5, 3], bits[6, 4], bits[7] = np.nan, np.inf, -np.inf
    got = grad(gpu, ids, bits, "f32", vocab, 0, width, 1.0, "f32")
    hit = {(int(ids[5, 0]), 3), (int(ids[6, 0]), 4)} | {(int(ids[7, 0]), j) for j in range(width)}
    odd = {tuple(int(v) for v in i) for i in np.argwhere(~np.isfinite(got))}
    assert odd == hit


def whole(rng, shape):
    """whole numbers but 0, whose sums are exact in any order while they are below 2^24"""
    return (rng.integers(1, 9, shape) * rng.choice([-1, 1], shape)).astype(np.float32)


def check_whole(gpu, ids, vocab, slot_rows, width, dtype, out, rng, dy_pad=0, pad=0):
    n, t = ids.shape
    bits, dy = R.to_bits(whole(rng, (n, width)), dtype)
    ref, size, count = SR.embed_grad(ids, dy, vocab, slot_rows, 0.25)
    assert size.max() < 2 ** 22
    for old in (None, R.to_bits(whole(rng, ref.shape), out)):
        want = R.to_bits(ref if old is None else ref + old[1], out)[0]
        got = grad(gpu, ids, bits, dtype, vocab, slot_rows, width, 0.25, out, dy_pad, pad, old=None if old is None else old[0])
        assert np.array_equal(R.from_bits(np.ascontiguousarray(got)), R.from_bits(want))
    return count


@pytest.mark.parametrize("n,t,vocab,slot_rows,width,dtype,out,how,dy_pad,pad", GRADS)
def test_gradient_of_whole_numbers(gpu, n, t, vocab, slot_rows, width, dtype, out, how, dy_pad, pad):
    """equal, so that no position of a frequent row is lost or taken twice"""
    rng = np.random.default_rng([n, t, vocab, width, 1])
    check_whole(gpu, make_ids(rng, n, t, vocab, how), vocab, slot_rows, width, dtype, out, rng, dy_pad, pad)


@pytest.mark.parametrize("counts,rows,vocab", [
    ((65,), 500, 500), ((65,), 500, 40000), ((65,), 1000, 1000), ((65,), 1100, 2000003), ((33,), 900, 700000), ((65,), 16000, 16000),
    ((1, 31, 32, 33, 63, 64, 65, 66, 127, 128, 129, 193, 4095, 4096, 4097, 8193), 1, 50),
    ((1, 31, 32, 33, 63, 64, 65, 66, 127, 128, 129, 193, 4095, 4096, 4097, 8193), 4, 5000),
    ((129, 65, 64, 2), 9000, 50000)])
@pytest.mark.parametrize("width,out", [(4, "f32"), (41, "bf16")])
def test_rows_of_so_many_ids(gpu, counts, rows, vocab, width, out):
    """rows of exactly as many ids as one chunk, two or more begin at; all ids in cut rows"""
    rng = np.random.default_rng([sum(counts), rows, vocab, width])
    n = sum(counts) * rows
    names = rng.permutation(vocab)[:rows * len(counts)]
    ids = np.repeat(names, np.tile(counts, rows))
    assert len(ids) == n
    ids = ids[rng.permutation(n)].astype(np.int32)[:, None]
    got = check_whole(gpu, ids, vocab, 0, width, "f32", out, rng)
    assert set(got[got > 0]) == set(counts)
