"""The scoring and training entry points refuse what they cannot take before
anything is launched (no GPU needed: no pointer below is looked at)."""
import ctypes
import math

import numpy as np
import pytest

P = 4096  # an aligned address that is never read


@pytest.fixture(scope="module")
def d3s():
    import d3s
    d3s.lib()
    return d3s


SCORE = dict(logits=P, dtype=0, n_rows=4, vocab=100, row_stride=100, temperature=1.0, banned=None, tokens=P, n_tokens=1,
             logprobs=P)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), -4), (dict(n_rows=-1), -1), (dict(n_rows=1 << 31), -1), (dict(vocab=0), -1),
    (dict(vocab=1 << 24, row_stride=1 << 24), -2), (dict(row_stride=99), -1), (dict(n_tokens=-1), -1),
    (dict(n_tokens=65), -1), (dict(n_top=-1), -1), (dict(n_top=65), -1), (dict(vocab=10, row_stride=10, n_top=11), -1),
    (dict(logits=None), -1), (dict(logits=P + 2), -1), (dict(dtype=1, logits=P + 1), -1), (dict(tokens=None), -1),
    (dict(n_rows=0), 0), (dict(n_rows=0, logits=None, tokens=None), 0)])
def test_logprob(d3s, change, status):
    assert d3s.logprob_raw(**{**SCORE, **change}) == status


def test_logprob_workspace(d3s):
    size = d3s.lib().d3s_logprob_workspace_bytes
    assert size(1, 4096, 4097, 0) == 0  # rows enough: one workgroup each
    need = size(1, 64, 151936, 20)
    assert need > 0
    assert size(5, 1, 10, 0) == -4 and size(0, 1, 0, 0) == -1 and size(0, 1, 10, 11) == -1
    assert size(0, -1, 10, 0) == -1 and size(0, 1, 1 << 24, 0) == -2
    base = dict(SCORE, dtype=1, n_rows=64, vocab=151936, row_stride=151936, n_top=20, top_ids=P)
    assert d3s.logprob_raw(**base, workspace=(P, need - 1)) == -7
    assert d3s.logprob_raw(**base, workspace=(None, need)) == -7
    assert d3s.logprob_raw(**base, workspace=(P, -1)) == -1
    assert d3s.logprob_raw(**base, workspace=(P + 4, need)) == -1  # not 256-byte aligned


GRAD = dict(logits=P, dtype=0, n_rows=4, vocab=100, row_stride=100, temperature=1.0, banned=None, tokens=P, n_tokens=1,
            row_stats=P, entropy=P, grad_logprobs=P, grad_entropy=P, grad_logits=2 * P, grad_row_stride=100)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(n_rows=-1), -1), (dict(vocab=0), -1), (dict(vocab=1 << 24, row_stride=1 << 24), -2),
    (dict(row_stride=99), -1), (dict(grad_row_stride=99), -1), (dict(n_tokens=65), -1), (dict(logits=None), -1),
    (dict(row_stats=None), -1), (dict(grad_logits=None), -1), (dict(grad_logits=P + 2), -1), (dict(tokens=None), -1),
    (dict(grad_logprobs=None), -1), (dict(entropy=None), -1), (dict(grad_logits=P, grad_row_stride=128), -1),
    (dict(n_rows=0), 0)])
def test_logprob_backward(d3s, change, status):
    assert d3s.logprob_backward_raw(**{**GRAD, **change}) == status


DENSE = dict(x=P, x_stride=64, w=P, w_stride=64, m=8, n=32, k=64, y=P, y_stride=32, y_dtype=1)


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), -1), (dict(n=-1), -1), (dict(k=-1), -1), (dict(m=1 << 31), -1), (dict(x_stride=63), -1),
    (dict(w_stride=63), -1), (dict(x_transposed=True, x_stride=7), -1), (dict(w_transposed=True, w_stride=31), -1),
    (dict(y_stride=31), -1), (dict(residual=P, residual_stride=31), -1), (dict(z=P, z_stride=31), -1),
    (dict(y_dtype=4), -4), (dict(activation=-1), -1), (dict(activation=5), -1), (dict(x=None), -1), (dict(w=None), -1),
    (dict(y=None), -1), (dict(x=P + 1), -1), (dict(w=P + 1), -1), (dict(y=P + 1), -1), (dict(y=P + 2, y_dtype=0), -1),
    (dict(bias=P + 1), -1), (dict(z=P + 1, z_stride=32), -1), (dict(residual=P + 1, residual_stride=32), -1),
    (dict(m=0), 0), (dict(n=0, w=None, y=None), 0)])
def test_dense(d3s, change, status):
    assert d3s.dense_raw(**{**DENSE, **change}) == status


def test_dense_null(d3s):
    assert d3s.lib().d3s_dense_bf16(None, None) == -1
    assert d3s.lib().d3s_dense_workspace_bytes(None) == -1
    p = d3s.dense_params(**dict(DENSE, y_dtype=9))
    assert d3s.lib().d3s_dense_workspace_bytes(ctypes.byref(p)) == -4


ACT = dict(dy=P, dy_stride=32, z=P, z_stride=32, m=8, n=32, activation=2, dz=2 * P, dz_stride=32, dbias=P)


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), -1), (dict(n=1 << 31), -1), (dict(activation=5), -1), (dict(dy_stride=31), -1),
    (dict(z_stride=31), -1), (dict(dz_stride=31), -1), (dict(dy=None), -1), (dict(z=None), -1), (dict(dy=P + 1), -1),
    (dict(z=P + 1), -1), (dict(dz=P + 1), -1), (dict(dbias=P + 2), -1), (dict(n=0), 0), (dict(dz=None, dbias=None), 0),
    (dict(m=0, dbias=None), 0)])
def test_activation_backward(d3s, change, status):
    assert d3s.dense_activation_backward_raw(**{**ACT, **change}) == status


def test_clip(d3s):
    src = np.array([P, 2 * P], np.uint64)
    n = np.array([10, 20], np.int64)
    dt = np.array([0, 1], np.int32)

    def call(src=src, dst=src, numel=n, dtypes=dt, n_tensors=2, max_norm=1.0, norm=P, **kw):
        at = lambda a: None if a is None else a.ctypes.data  # noqa: E731
        return d3s.clip_grads_raw(at(src), at(dst), at(numel), at(dtypes), n_tensors, max_norm, norm, **kw)

    assert call(n_tensors=-1) == -1 and call(norm=None) == -1 and call(norm=P + 2) == -1
    for bad in (0.0, -1.0, math.nan):
        assert call(max_norm=bad) == -1
    assert call(src=None) == -1 and call(numel=None) == -1 and call(dtypes=None) == -1
    assert call(dtypes=np.array([0, 2], np.int32)) == -4
    assert call(numel=np.array([10, -1], np.int64)) == -1
    assert call(src=np.array([P, 0], np.uint64)) == -1 and call(dst=np.array([P, 0], np.uint64)) == -1
    assert call(src=np.array([P + 2, P], np.uint64)) == -1 and call(dst=np.array([P, P + 1], np.uint64)) == -1
    need = d3s.lib().d3s_clip_grads_workspace_bytes(2)
    assert need > 0 and d3s.lib().d3s_clip_grads_workspace_bytes(-1) == -1
    assert call(workspace=(P, need - 1)) == -7 and call(workspace=(P + 8, need)) == -1
