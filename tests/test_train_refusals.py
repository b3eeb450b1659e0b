"""More of what the scoring and training entry points refuse, and what their
workspace queries promise (no GPU needed: no pointer below is looked at)."""
import pytest

P = 4096  # an aligned address that is never read


@pytest.fixture(scope="module")
def d3s():
    import d3s
    d3s.lib()
    return d3s


@pytest.mark.parametrize("y_dtype", [0, 1])
@pytest.mark.parametrize("residual_stride", [32, 41, 100])
def test_dense_in_place_at_another_stride(d3s, y_dtype, residual_stride):
    """a residual that is y itself lies where y does: at another stride one workgroup's
    outputs would be rows that another has yet to read"""
    call = dict(x=P, x_stride=64, w=P, w_stride=64, m=8, n=32, k=64, y=2 * P, y_stride=40, y_dtype=y_dtype,
                residual=2 * P, residual_stride=residual_stride)
    assert d3s.dense_raw(**call) == -1
    assert d3s.dense_raw(**call, workspace=(P, 1 << 30)) == -1
    assert d3s.dense_raw(**dict(call, m=2)) == -1


@pytest.mark.parametrize("dz_stride", [32, 41, 100])
def test_activation_gradient_in_place_at_another_stride(d3s, dz_stride):
    """the same of a dz that is dy itself"""
    call = dict(dy=P, dy_stride=40, z=2 * P, z_stride=32, m=8, n=32, activation=2, dz=P, dz_stride=dz_stride, dbias=3 * P)
    assert d3s.dense_activation_backward_raw(**call) == -1
    assert d3s.dense_activation_backward_raw(**dict(call, dbias=None)) == -1
    assert d3s.dense_activation_backward_raw(**call, workspace=(P, 1 << 30)) == -1
    assert d3s.dense_activation_backward_raw(**dict(call, m=2, z=None, activation=0)) == -1


@pytest.mark.parametrize("dtype", [0, 1])
def test_scores_workspace_covers_a_call_without_alternatives(d3s, dtype):
    """n_top with neither top_ids nor top_logprobs is a call without alternatives,
    which is cut into other segments: what was queried with n_top serves it too"""
    size = d3s.lib().d3s_logprob_workspace_bytes
    for rows in (1, 2, 7, 64, 500, 1024, 2048, 2049):
        for vocab in (64, 4097, 8185, 16384, 60000, 151936, 1000003):
            for n_top in (1, 5, 20, 64):
                assert size(dtype, rows, vocab, n_top) >= size(dtype, rows, vocab, 0), (rows, vocab, n_top)
