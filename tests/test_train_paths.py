"""Dense layers, their gradients and clipping where work is split and joined: the
same bits at every call and on every stream, captured and replayed, the plan's
edges (rows peeled from large tiles, split sums, short inner lengths)."""
import ctypes

import numpy as np
import pytest

import train_ref as R
import test_clip as C
import test_score as S
from test_dense import product, slopes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    import d3s
    import hiprt
    d3s.lib()
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    return d3s


# (m, n, k, x by the inner index, w by it): split tiles, split few rows, rows peeled, rounds
SPLIT = [(256, 2048, 4096, False, False), (200, 600, 3001, False, False), (16, 1024, 4096, False, True),
         (1, 640, 8192, True, True), (300, 512, 2000, True, True), (48, 2048, 2048, False, False),
         (129, 130, 5000, False, True)]


class Call:
    def __init__(self, gpu, D, shape, seed=0, own_workspace=False):
        m, n, k, xt, wt = shape
        rng = np.random.default_rng([m, n, k, seed])
        self.gpu, self.shape = gpu, shape
        self.x = D.put(R.to_bits(rng.standard_normal((k, m) if xt else (m, k)), "bf16")[0])
        self.w = D.put(R.to_bits(rng.standard_normal((k, n) if wt else (n, k)) * k ** -0.5, "bf16")[0])
        self.y = D.room(4 * m * n, 0xee)
        self.ws = None
        if own_workspace:
            p = gpu.dense_params(**self.args())
            W = gpu.Workspace(gpu.lib().d3s_dense_workspace_bytes(ctypes.byref(p)))
            D.held.append(W.buf)
            self.ws = W.arg()

    def args(self):
        m, n, k, xt, wt = self.shape
        return dict(x=self.x.ptr, x_stride=m if xt else k, w=self.w.ptr, w_stride=n if wt else k, m=m, n=n, k=k,
                    y=self.y.ptr, y_stride=n, y_dtype=self.gpu.DTYPE_F32, x_transposed=xt, w_transposed=wt)

    def run(self, stream=None):
        assert self.gpu.dense_raw(**self.args(), stream=stream, workspace=self.ws) == 0

    def out(self):
        m, n = self.shape[:2]
        return self.y.download((m, n), np.uint32)


@pytest.mark.parametrize("shape", SPLIT)
def test_the_same_bits_each_time(gpu, shape):
    import hiprt
    with R.Arena() as D:
        c = Call(gpu, D, shape)
        own = Call(gpu, D, shape, own_workspace=True)
        c.run()
        hiprt.synchronize()
        first = c.out()
        for _ in range(4):
            c.run()
            own.run()
            hiprt.synchronize()
            assert np.array_equal(c.out(), first) and np.array_equal(own.out(), first)


def test_two_streams_at_once(gpu):
    import hiprt
    streams = [hiprt.Stream(), hiprt.Stream()]
    with R.Arena() as D:
        calls = [[Call(gpu, D, s, seed) for s in SPLIT] for seed in (1, 2)]
        for group in calls:
            for c in group:
                c.run()
        hiprt.synchronize()
        want = [[c.out() for c in group] for group in calls]
        for c in calls[0] + calls[1]:
            c.y.upload(np.zeros(c.y.nbytes, np.uint8))
        for _ in range(3):
            for pair in zip(*calls):
                for s, c in zip(streams, pair):
                    c.run(s.ptr)
        hiprt.synchronize()
        for group, refs in zip(calls, want):
            for c, ref in zip(group, refs):
                assert np.array_equal(c.out(), ref)
    for s in streams:
        assert gpu.lib().d3s_stream_workspace_release(s.ptr) == 0
        s.destroy()


def test_captured_and_replayed(gpu):
    """products with split sums, an activation's gradient with column sums and
    clipping in one graph, with other work on their workspaces between replays"""
    import hiprt
    H = hiprt.hip()
    s = hiprt.Stream()
    rng = np.random.default_rng(5)
    m, n = 500, 300
    with R.Arena() as D:
        calls = [Call(gpu, D, shape, 3, own_workspace=True) for shape in SPLIT[:4]]
        dy, z, dz, db = D.room(2 * m * n), D.room(2 * m * n), D.room(2 * m * n), D.room(4 * n)
        g, out, norm = D.room(4 * 5000), D.room(4 * 5000), D.room(4)
        src, dst = np.array([g.ptr, g.ptr + 4 * 3000], np.uint64), np.array([out.ptr, out.ptr + 4 * 3000], np.uint64)
        numel, dt = np.array([3000, 2000], np.int64), np.zeros(2, np.int32)
        W1 = gpu.Workspace(gpu.lib().d3s_dense_activation_backward_workspace_bytes(m, n, 1))
        W2 = gpu.Workspace(gpu.lib().d3s_clip_grads_workspace_bytes(2))
        D.held += [W1.buf, W2.buf]
        hiprt.synchronize()

        def work(stream, ws=True):
            for c in calls:
                c.run(stream)
            rc = gpu.dense_activation_backward_raw(dy.ptr, n, z.ptr, n, m, n, 2, dz.ptr, n, db.ptr, stream=stream,
                                                   workspace=W1.arg() if ws else None)
            return rc or gpu.clip_grads_raw(src.ctypes.data, dst.ctypes.data, numel.ctypes.data, dt.ctypes.data, 2, 0.5,
                                            norm.ptr, stream=stream, workspace=W2.arg() if ws else None)

        graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
        hiprt.check(H.hipStreamBeginCapture(s.ptr, 2))
        refused = gpu.clip_grads_raw(src.ctypes.data, dst.ctypes.data, numel.ctypes.data, dt.ctypes.data, 2, 0.5, norm.ptr,
                                     stream=s.ptr)
        rc = work(s.ptr)
        hiprt.check(H.hipStreamEndCapture(s.ptr, ctypes.byref(graph)))
        assert refused == -7 and rc == 0
        assert set(hiprt.graph_node_types(graph)) == {"kernel"}
        hiprt.check(H.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0))

        def results():
            return [c.out() for c in calls] + [dz.download((m, n), np.uint16), db.download((n,), np.uint32),
                                               out.download((5000,), np.uint32), norm.download((1,), np.uint32)]

        for i in range(4):
            for b in (dy, z):
                b.upload(R.to_bits(rng.standard_normal((m, n)), "bf16")[0])
            g.upload(rng.standard_normal(5000).astype(np.float32))
            for c in calls:
                c.x.upload(R.to_bits(rng.standard_normal(c.x.nbytes // 2), "bf16")[0])
            hiprt.synchronize()
            hiprt.check(H.hipGraphLaunch(ex, s.ptr))
            s.synchronize()
            replayed = results()
            assert work(s.ptr) == 0  # eagerly, on the same workspaces
            s.synchronize()
            for a, b in zip(replayed, results()):
                assert np.array_equal(a, b), i
        H.hipGraphExecDestroy(ex)
        H.hipGraphDestroy(graph)
        s.destroy()


@pytest.mark.parametrize("xt,wt", [(False, False), (False, True), (True, False), (True, True)])
def test_plans(gpu, xt, wt):
    """rows that a large tile would leave nearly empty, several rounds of tiles,
    inner lengths of a stage more or less, short rows by the inner index"""
    product(gpu, 2049, 2048, 200, xt, wt, residual=True, out="f32")
    product(gpu, 2080, 1030, 136, xt, wt, bias=True, act="gelu_tanh", keep=True, residual=True)
    for k in (63, 64, 65, 127, 128, 129, 191, 193):
        product(gpu, 130, 260, k, xt, wt)
    for m, n in ((100, 3), (100, 5), (100, 7), (70, 9), (33, 2), (65, 1)):
        product(gpu, m, n, 100, xt, wt, residual=True, in_place=True)
        product(gpu, m, n, 64, xt, wt, offset=1)


def test_large_tiles_with_everything(gpu):
    product(gpu, 2304, 2304, 192, bias=True, act="gelu", residual=True, keep=True)
    product(gpu, 2304, 2200, 200, bias=True, act="silu", residual=True, keep=True, pads=(0, 0, 8))
    product(gpu, 2304, 2200, 201, act="relu", residual=True, out="f32", pads=(3, 1, 1))
    product(gpu, 2304, 2304, 136, False, True, residual=True, pads=(0, 0, 0))
    product(gpu, 2304, 2304, 136, True, False, residual=True, out="f32")
    product(gpu, 2304, 2304, 136, True, True, residual=True, out="f32", in_place=True)


def test_wide_activation_gradients(gpu):
    slopes(gpu, 3, 9000, "gelu")
    slopes(gpu, 20000, 3, "silu", pads=(1, 0, 2))


def test_infinite_activations(gpu):
    """what an activation and its slope make of infinities and NaN"""
    import hiprt
    inf, nan = np.inf, np.nan
    x = np.float32([[inf, -inf, nan, 1.0]]).T  # m = 4, k = 1
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        with R.Arena() as D:
            xb, wb = R.to_bits(x, "bf16")[0], R.to_bits(np.ones((1, 1)), "bf16")[0]
            y, dz = D.room(16), D.room(8)
            X = D.put(xb)
            assert gpu.dense_raw(X.ptr, 1, D.put(wb).ptr, 1, 4, 1, 1, y.ptr, 1, gpu.DTYPE_F32,
                                 activation=gpu.ACTIVATIONS[act]) == 0
            one = D.put(R.to_bits(np.ones((4, 1)), "bf16")[0])
            assert gpu.dense_activation_backward_raw(one.ptr, 1, X.ptr, 1, 4, 1, gpu.ACTIVATIONS[act], dz.ptr, 1, None) == 0
            hiprt.synchronize()
            got, d = y.download((4,), np.float32), R.from_bits(dz.download((4,), np.uint16))
        assert got[0] == inf and got[1] == 0 and np.isnan(got[2]), (act, got)
        assert d[0] == 1 and d[1] == 0 and np.isnan(d[2]), (act, d)


@pytest.mark.parametrize("xt,wt", [(False, False), (False, True), (True, False), (True, True)])
def test_outputs_peeled(gpu, xt, wt):
    """outputs, and rows and outputs, that a last tile would leave nearly empty"""
    product(gpu, 4096, 4097, 130, xt, wt, bias=True, act="silu", keep=True, residual=True)
    product(gpu, 4096, 2070, 136, xt, wt, residual=True, out="f32", in_place=True)
    product(gpu, 4097, 4098, 97, xt, wt, bias=True, residual=True, pads=(1, 1, 3), offset=1)


@pytest.mark.parametrize("m,n,k", [(9, 513, 1025), (1, 4097, 4097), (33, 200, 999), (64, 300, 513)])
def test_few_rows_at_any_element(gpu, m, n, k):
    for xt, wt in ((False, False), (False, True), (True, False)):
        product(gpu, m, n, k, xt, wt, bias=True, act="gelu", residual=True)
        product(gpu, m, n, k, xt, wt, pads=(2, 1, 0), offset=1, out="f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,V,top,pad,offset", [(700, 10001, 33, 0, 0), (130, 60003, 64, 1, 3), (1025, 8200, 2, 0, 1)])
def test_alternatives_of_long_segments(gpu, n, V, top, pad, offset, dtype):
    """so many rows that a segment is more than is held at once: it is read again for
    the alternatives, several times where there are more ties than are filed"""
    rng = np.random.default_rng([n, V])
    x = rng.standard_normal((n, V), np.float32) * 2.5
    x[1::8] = 0
    x[2::8] = rng.integers(0, 2, x[2::8].shape)
    x[3::8] = np.round(x[3::8])
    x[4::8, : V - 5] = -np.inf
    x[5] = -np.inf
    x[6, V - 1] = np.nan
    bits, l = R.to_bits(x, dtype)
    tokens = rng.integers(0, V, (n, 1))
    banned = np.where(rng.random(n) < 0.5, l.argmax(1), -1)
    S.check(S.run(gpu, bits, 0.8, banned, tokens, top, pad, offset), R.score(l, S.temperatures(0.8, n), banned, tokens, top))


@pytest.mark.parametrize("sizes", [[3] * 248, [3] * 249, [0, 7] * 260, list(range(1, 500)) + [300000, 0, 70001] + [9] * 300,
                                   [1, 2, 8] * 1366, [5] * 4160 + [100000] + [2] * 4160])
def test_many_tensors(gpu, sizes):
    """more tensors than travel with one launch, with every number of 64s and of 4096s of them"""
    t = C.tensors_of(sizes)
    norm = float(np.sqrt(sum(float((R.from_bits(b) ** 2).sum()) for b, _ in t)))
    for limit in (norm / 3, norm * 2):
        limit = float(np.float32(limit))
        C.check(*C.run(gpu, t, limit, shift=3, use_ws=True), t, limit)
        C.check(*C.run(gpu, t, limit, in_place=True), t, limit)
    n, _ = C.run(gpu, t, 1.0, norm_only=True)
    C.check(n, [], t, 1.0)


@pytest.mark.parametrize("xt,wt", [(False, False), (False, True), (True, False), (True, True)])
def test_last_round_of_tiles_apart(gpu, xt, wt):
    """outputs or rows whose tiles would begin one more round of the whole chip are a product of their own"""
    product(gpu, 1500, 11008, 130, xt, wt, bias=True, act="silu", keep=True, residual=True)
    product(gpu, 11008, 1500, 70, xt, wt, bias=True, act="gelu", keep=True, residual=True, out="f32", in_place=True)
    product(gpu, 11010, 1501, 65, xt, wt, bias=True, keep=True, residual=True, pads=(1, 1, 3), offset=1)
    product(gpu, 1537, 11011, 200, xt, wt, residual=True, out="f32")
