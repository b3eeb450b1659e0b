"""The operators between ids and logits where calls meet: the same bits at every call, two
streams at once, captured and replayed, one workspace for all of them, rows far
apart, more work than a launch's workgroups."""
import ctypes

import numpy as np
import pytest

import step_ref as SR
import train_ref as R
import test_dropout as TD
import test_embed as TE
import test_norm as TN
import test_verify as TV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


class Verify:
    """long rows: two launches that leave sums in a workspace"""

    def __init__(self, gpu, D, seed, n=12, L=3, V=40000):
        self.gpu, self.shape = gpu, (n, L, V)
        target, draft, self.drafted, self.ua, self.ud, _ = TV.inputs(n, L, V, seed)
        tb, self.tv = R.to_bits(target.reshape(-1, V), "bf16")
        db, self.dv = R.to_bits(draft.reshape(-1, V), "bf16")
        self.tv, self.dv = self.tv.reshape(n, L + 1, V), self.dv.reshape(n, L, V)
        self.ua = SR.keep_off_borders(self.tv, self.dv, self.drafted, np.ones(n), np.ones(n), self.ua)
        self.tokens, self.acc = D.room(4 * n * (L + 1), 0x55), D.room(4 * n, 0x55)
        self.args = dict(target=D.put(tb).ptr, target_dtype=1, target_stride=V, draft=D.put(db).ptr, draft_dtype=1,
                         draft_stride=V, n_seqs=n, n_draft=L, vocab=V, drafted=D.put(self.drafted.astype(np.int32)).ptr,
                         lengths=None, temperature=1.0, draft_temperature=1.0, u_accept=D.put(self.ua).ptr,
                         u_draw=D.put(self.ud).ptr, tokens=self.tokens.ptr, n_accepted=self.acc.ptr)

    def need(self):
        return self.gpu.lib().d3s_verify_workspace_bytes(ctypes.byref(self.gpu.verify_params(**self.args)))

    def run(self, stream=None, ws=None):
        return self.gpu.verify_raw(**self.args, stream=stream, workspace=ws)

    def out(self):
        n, L, _ = self.shape
        return [self.tokens.download((n, L + 1), np.int32), self.acc.download((n,), np.int32)]

    def check(self):
        n = self.shape[0]
        ref = SR.verify(self.tv, self.dv, self.drafted, None, np.ones(n), np.ones(n), self.ua, self.ud)
        got = self.out()
        assert np.array_equal(got[0], ref[0]) and np.array_equal(got[1], ref[1])


class EmbedGrad:
    """frequent rows, cut into chunks that the last to arrive joins"""

    def __init__(self, gpu, D, seed, n=3000, t=2, vocab=500, width=136):
        self.gpu, self.shape = gpu, (n, t, vocab, width)
        rng = np.random.default_rng([seed, n])
        self.ids = TE.make_ids(rng, n, t, vocab, "zipf")
        self.bits, self.dy = R.to_bits(rng.standard_normal((n, width)), "bf16")
        self.idb, self.dyb, self.grad = D.put(self.ids), D.put(self.bits), D.room(4 * vocab * width, 0x55)

    def need(self):
        n, t, vocab, width = self.shape
        return self.gpu.lib().d3s_embed_backward_workspace_bytes(n, t, vocab, 0, width)

    def run(self, stream=None, ws=None):
        n, t, vocab, width = self.shape
        return self.gpu.embed_backward_raw(self.idb.ptr, n, t, self.dyb.ptr, 1, width, vocab, 0, width, 1.0, 0, self.grad.ptr, 0,
                                           width, stream=stream, workspace=ws)

    def out(self):
        _, _, vocab, width = self.shape
        return [self.grad.download((vocab, width), np.uint32)]

    def check(self):
        _, _, vocab, _ = self.shape
        ref, size, count = SR.embed_grad(self.ids, self.dy, vocab, 0, 1.0)
        assert count.max() > 300
        R.assert_near(self.out()[0].view(np.float32), ref, SR.U * (count[:, None] + 3) * size)


class NormGrad:
    """column sums of many workgroups"""

    def __init__(self, gpu, D, seed, n=5000, width=264):
        self.gpu, self.shape = gpu, (n, width)
        rng = np.random.default_rng([seed, n])
        (db, self.dy), (hb, self.h) = (R.to_bits(rng.standard_normal((n, width)), "bf16") for _ in range(2))
        self.rstd = (1 / np.sqrt((self.h ** 2).mean(1))).astype(np.float32)
        self.bufs = [D.put(db), D.put(hb), D.put(self.rstd), D.room(2 * n * width, 0x55), D.room(4 * width, 0x55)]

    def need(self):
        return self.gpu.lib().d3s_rms_norm_backward_workspace_bytes(*self.shape, 1)

    def run(self, stream=None, ws=None):
        n, width = self.shape
        d, h, r, dx, dg = (b.ptr for b in self.bufs)
        return self.gpu.rms_norm_backward_raw(d, 1, width, h, width, None, r, None, 0, n, width, dx, width, dg, stream=stream,
                                              workspace=ws)

    def out(self):
        n, width = self.shape
        return [self.bufs[3].download((n, width), np.uint16), self.bufs[4].download((width,), np.uint32)]

    def check(self):
        n, width = self.shape
        ref, err, ref_g, size = SR.norm_grad(self.dy, self.h, np.ones(width), self.rstd.astype(np.float64), None)
        dx, dg = self.out()
        R.assert_near(R.from_bits(dx), ref, err + SR.BF16 * np.abs(ref) * 1.01)
        R.assert_near(dg.view(np.float32), ref_g, SR.U * (n + 4) * size)


KINDS = [Verify, EmbedGrad, NormGrad]


def equal(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_bits_each_time(gpu, kind):
    import hiprt
    with R.Arena() as D:
        c = kind(gpu, D, 1)
        W = gpu.Workspace(c.need())
        D.held.append(W.buf)
        assert c.run() == 0
        hiprt.synchronize()
        first = c.out()
        c.check()
        for _ in range(4):
            for ws in (None, W.arg()):
                assert c.run(ws=ws) == 0
                hiprt.synchronize()
                assert equal(c.out(), first)
        # the counters are left at zero
        assert (W.buf.download((65536,), np.uint32) == 0).all()


def test_two_streams_at_once(gpu):
    import hiprt
    streams = [hiprt.Stream(), hiprt.Stream()]
    with R.Arena() as D:
        calls = [[k(gpu, D, seed) for k in KINDS] for seed in (2, 3)]
        for group in calls:
            for c in group:
                assert c.run() == 0
        hiprt.synchronize()
        want = [[c.out() for c in group] for group in calls]
        for _ in range(3):
            for pair in zip(*calls):
                for s, c in zip(streams, pair):
                    assert c.run(s.ptr) == 0
        hiprt.synchronize()
        for group, refs in zip(calls, want):
            for c, ref in zip(group, refs):
                assert equal(c.out(), ref)
                c.check()
    for s in streams:
        assert gpu.lib().d3s_stream_workspace_release(s.ptr) == 0
        s.destroy()


def test_one_workspace_for_all(gpu):
    """calls of every kind in turn, with the sampler's and the score's, on one workspace"""
    import hiprt
    rng = np.random.default_rng(4)
    n, V = 4, 20000
    logits = (rng.standard_normal((n, V)) * 2).astype(np.float32)
    u = (rng.integers(0, 1 << 24, (n, 30)) * 2.0 ** -24).astype(np.float32)
    want = gpu.sample(logits, u, 1.0, 0.9)["ids"]
    with R.Arena() as D:
        calls = [k(gpu, D, 5) for k in KINDS]
        need = max([c.need() for c in calls] + [gpu.workspace_bytes(0, n, V, 30), gpu.lib().d3s_logprob_workspace_bytes(0, n, V, 5)])
        W = gpu.Workspace(need)
        lb, ub, ids, top = D.put(logits), D.put(u), D.room(4 * n), D.room(4 * n * 5)
        D.held.append(W.buf)
        for _ in range(3):
            for c in calls:
                assert c.run(ws=W.arg()) == 0
                assert gpu.sample_raw(lb.ptr, 0, n, V, V, ub.ptr, 30, 1.0, 0.9, None, ids.ptr, workspace=W.arg()) == 0
                assert gpu.logprob_raw(lb.ptr, 0, n, V, V, 1.0, None, None, 0, None, n_top=5, top_ids=top.ptr, workspace=W.arg()) == 0
            hiprt.synchronize()
            for c in calls:
                c.check()
            assert np.array_equal(ids.download((n,), np.int32), want)
            assert np.array_equal(top.download((n, 5), np.int32), np.argsort(-logits, 1, kind="stable")[:, :5])


def test_captured_and_replayed(gpu):
    """all in one graph on workspaces of the caller's, replayed with the same calls made eagerly between; a
    captured dropout drops other elements at every replay by its device counter"""
    import hiprt
    H = hiprt.hip()
    s = hiprt.Stream()
    rng = np.random.default_rng(6)
    with R.Arena() as D:
        calls = [k(gpu, D, 7) for k in KINDS]
        spaces = [gpu.Workspace(c.need()) for c in calls]
        D.held += [w.buf for w in spaces]
        x = D.put(np.ones((9, 333), np.float32))
        y, add = D.room(4 * 9 * 333), D.put(np.zeros(1, np.uint64))
        table, ids, row = D.put(rng.standard_normal((50, 64)).astype(np.float32)), D.put(np.arange(6, dtype=np.int32)), D.room(4 * 2 * 64)
        z, rstd, q, scales = D.room(4 * 2 * 64), D.room(8), D.room(2 * 64), D.room(4 * 2 * 2)
        cand, probs = TV.ranked_rows(3 * 2, 30, 100, rng)
        cb, pb, dr = D.put(cand), D.put(probs), D.put(cand.reshape(3, 2, 30)[:, 0, :1].copy())
        ua, ud, tok, acc = D.put(np.full((3, 1), 0.5, np.float32)), D.put(rng.random((3, 30)).astype(np.float32)), D.room(24), D.room(12)
        hiprt.synchronize()

        def work(stream, ws=True):
            rc = [c.run(stream, w.arg() if ws else None) for c, w in zip(calls, spaces)]
            rc.append(gpu.dropout_raw(x.ptr, 0, 333, None, 0, 9, 333, 0.5, 11, 100, add.ptr, y.ptr, 333, stream=stream))
            rc.append(gpu.embed_raw(ids.ptr, 2, 3, table.ptr, 0, 64, 50, 0, 64, 1.0, row.ptr, 0, 64, stream=stream))
            rc.append(gpu.rms_norm_raw(row.ptr, 0, 64, None, 0, None, 0, None, 1e-6, 2, 64, z.ptr, 0, 64, rstd=rstd.ptr, stream=stream))
            rc.append(gpu.rms_norm_raw(row.ptr, 0, 64, None, 0, None, 0, None, 1e-6, 2, 64, q.ptr, 2, 64, group=32, scales=scales.ptr,
                                       stream=stream))
            rc.append(gpu.verify_ranked_raw(cb.ptr, pb.ptr, 30, None, None, 0, 3, 1, dr.ptr, None, ua.ptr, ud.ptr, tok.ptr, acc.ptr,
                                            stream=stream))
            return rc

        def results():
            return [a for c in calls for a in c.out()] + [y.download((9, 333), np.uint32), row.download((2, 64), np.uint32),
                                                          z.download((2, 64), np.uint32), q.download((2, 64), np.uint8),
                                                          scales.download((2, 2), np.uint32), tok.download((3, 2), np.int32),
                                                          acc.download((3,), np.int32)]

        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        hiprt.check(H.hipStreamBeginCapture(s.ptr, 2))
        refused = [c.run(s.ptr) for c in calls]  # no block of the stream's in a graph
        rc = work(s.ptr)
        hiprt.check(H.hipStreamEndCapture(s.ptr, ctypes.byref(graph)))
        assert refused == [-7] * len(calls) and rc == [0] * 8
        assert set(hiprt.graph_node_types(graph)) == {"kernel"}
        hiprt.check(H.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0))
        masks = []
        for i in range(4):
            add.upload(np.array([i], np.uint64))
            for b in (calls[1].dyb, calls[2].bufs[0]):
                n = b.nbytes // 2
                b.upload(R.to_bits(rng.standard_normal(n), "bf16")[0])
            hiprt.synchronize()
            hiprt.check(H.hipGraphLaunch(ex, s.ptr))
            s.synchronize()
            replayed = results()
            masks.append(replayed[-7])
            assert work(s.ptr) == [0] * 8  # eagerly, on the same workspaces
            s.synchronize()
            assert equal(replayed, results()), i
        calls[0].check()
        assert all(not np.array_equal(masks[0], m) for m in masks[1:])
        H.hipGraphExecDestroy(ex)
        H.hipGraphDestroy(graph)
        s.destroy()


def test_rows_past_32_bits(gpu):
    """rows whose offsets pass 2^32 bytes and 2^32 elements"""
    import hiprt
    if hiprt.free_memory() < 60 << 30:
        pytest.skip("not enough memory")
    S = (1 << 31) + 24  # elements from one row to the next
    rng = np.random.default_rng(8)
    n, width = 3, 200
    bits, v = R.to_bits(rng.standard_normal((n, width)), "bf16")
    put = lambda b, rows: [b.upload(r, offset=2 * S * i) for i, r in enumerate(rows)]  # noqa: E731
    get = lambda b: np.stack([b.download((width,), np.uint16, offset=2 * S * i) for i in range(n)])  # noqa: E731
    with R.Arena() as D:
        a, b = D.room(2 * (2 * S + width)), D.room(2 * (2 * S + width))
        put(a, bits)
        assert gpu.rms_norm_raw(a.ptr, 1, S, None, 0, None, 0, None, 1e-6, n, width, b.ptr, 1, S) == 0
        hiprt.synchronize()
        y, _ = SR.norm(v, np.ones(width), 1e-6)
        R.assert_near(R.from_bits(get(b)), y, (SR.BF16 * 1.01 + SR.U * 20) * np.abs(y))
        assert gpu.dropout_raw(a.ptr, 1, S, None, 0, n, width, 0.5, 3, 4, None, b.ptr, S) == 0
        hiprt.synchronize()
        TD.check(get(b), v, None, "bf16", 0.5, 3, 4)
        ids = np.array([[2], [0], [1], [2]], np.int32)
        out = D.room(4 * 4 * width)
        assert gpu.embed_raw(D.put(ids).ptr, 4, 1, a.ptr, 1, S, n, 0, width, 1.0, out.ptr, 0, width) == 0
        hiprt.synchronize()
        assert np.array_equal(out.download((4, width), np.float32), v[ids[:, 0]].astype(np.float32))
        # dy [4] from the same place, the gradient S elements a row
        assert gpu.embed_backward_raw(D.put(np.array([[1], [2], [2]], np.int32)).ptr, 3, 1, a.ptr, 1, S, n, 0, width, 1.0, 0,
                                      b.ptr, 1, S) == 0
        hiprt.synchronize()
        got = R.from_bits(get(b))
        assert (got[0] == 0).all() and np.array_equal(got[1], v[0])
        R.assert_near(got[2], v[1] + v[2], (SR.BF16 * 1.01 + SR.U) * np.abs(v[1] + v[2]))


@pytest.mark.parametrize("vocab", [2000003, 5000000])
def test_wide_ranges_of_the_table(gpu, vocab):
    """many ids over a long table: ranges of more rows a workgroup; narrow rows"""
    rng = np.random.default_rng(9)
    n = 60000
    ids = TE.make_ids(rng, n, 1, vocab, "zipf")
    bits, dy = R.to_bits(rng.standard_normal((n, 4)), "f32")
    got = TE.grad(gpu, ids, bits, "f32", vocab, 0, 4, 1.0, "f32")
    ref, size, count = SR.embed_grad(ids, dy, vocab, 0, 1.0)
    R.assert_near(got, ref, SR.U * (count[:, None] + 3) * size)


def test_more_rows_than_workgroups(gpu):
    """2^21 and a few rows"""
    import hiprt
    n = (1 << 21) + 3
    rng = np.random.default_rng(10)
    bits, v = R.to_bits(rng.standard_normal((n, 3)), "f32")
    got, kept = TD.run(gpu, bits, None, "f32", 0.5, strides=(1, 0, 0)), None
    kept = TD.check(got, v, None, "f32", 0.5)
    assert abs(kept.mean() - 0.5) < 5 * 0.5 / np.sqrt(kept.size)
    y, rstd = SR.norm(v, np.ones(3), float(np.float32(1e-6)))
    f = TN.forward(gpu, bits, None, None, 1e-6, "f32", "f32", keep=False)
    R.assert_near(f["y"], y, SR.U * (SR.norm_steps(3) + 4) * np.abs(y) + 1e-38)
    # one sequence a row, no drafts: a draw from each
    with R.Arena() as D:
        u = (rng.integers(0, 1 << 24, n) * 2.0 ** -24).astype(np.float32)
        tok, acc = D.room(4 * n), D.room(4 * n)
        assert gpu.verify_raw(D.put(bits).ptr, 0, 3, None, 0, 0, n, 0, 3, None, None, 1.0, 1.0, None, D.put(u).ptr, tok.ptr, acc.ptr) == 0
        hiprt.synchronize()
        p = SR.probs(v, 1.0)
        c = p.cumsum(1)
        want = (c <= u[:, None].astype(np.float64) * c[:, -1:]).sum(1)
        assert np.array_equal(tok.download((n,), np.int32), want) and (acc.download((n,), np.int32) == 0).all()


@pytest.mark.parametrize("n,L,V", [(2049, 1, 16400), (2048, 0, 17000), (600, 3, 16385)])
def test_many_sequences_of_long_rows(gpu, n, L, V):
    """either side of the split's limits"""
    target, draft, drafted, ua, ud, _ = TV.inputs(n, L, V, 11) if L else (np.random.default_rng(1).standard_normal((n, 1, V)).astype(np.float32) * 2, np.zeros((n, 0, V), np.float32),
                                                                         np.zeros((n, 0), int), np.zeros((n, 0), np.float32), (np.arange(n) / n).astype(np.float32), None)
    TV.both(gpu, target, draft if L else None, drafted, None, 1.0, 1.0, ua, ud, "bf16", "bf16")


@pytest.mark.parametrize("n,L,V,certain", [(200, 2, 30011, False), (300, 1, 40001, True), (1030, 1, 9001, True), (1, 1, 3000017, False),
                                           (20, 2, 70007, True)])
def test_runs_of_a_block(gpu, n, L, V, certain):
    """blocks of one run and of several, the last ones past the row's end"""
    target, draft, drafted, ua, ud, _ = TV.inputs(n, L, V, 12)
    TV.both(gpu, target, None if certain else draft, drafted, None, 1.0, 1.0, ua, ud, "f32", "bf16")


@pytest.mark.parametrize("vocab,rows", [(2000003, 8000), (9000, 8000)])
def test_many_rows_that_are_cut(gpu, vocab, rows):
    """thousands of rows of fifty ids each, over a long table and over a short one: every call leaves
    the workspace's counters at zero"""
    import hiprt
    rng = np.random.default_rng([vocab, rows])
    n, width = 50 * rows, 4
    names = rng.permutation(vocab)[:rows]
    ids = names[rng.permutation(np.repeat(np.arange(rows), 50))].astype(np.int32).reshape(n, 1)
    bits, dy = R.to_bits(rng.standard_normal((n, width)), "f32")
    ref, size, count = SR.embed_grad(ids, dy, vocab, 0, 1.0)
    W = gpu.Workspace(gpu.lib().d3s_embed_backward_workspace_bytes(n, 1, vocab, 0, width))
    for _ in range(2):
        got = TE.grad(gpu, ids, bits, "f32", vocab, 0, width, 1.0, "f32", workspace=W.arg())
        R.assert_near(got, ref, SR.U * (count[:, None] + 3) * size)
        hiprt.synchronize()
        assert not W.buf.download((1 << 16,), np.uint32).any()
    W.buf.free()
