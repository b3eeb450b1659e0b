"""More of the log probabilities and their gradient: calls whose outputs are not
all wanted."""
import numpy as np
import pytest

import test_score as S
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


@pytest.mark.parametrize("n,V,top", [(1, 8185, 5), (1, 151936, 1), (3, 40001, 20), (700, 9000, 64)])
def test_alternatives_that_nobody_takes(gpu, n, V, top):
    """n_top with neither array of alternatives, in the workspace queried for n_top"""
    import hiprt
    rng, bits, l = S.make(n, V, "bf16", 11)
    tokens = rng.integers(0, V, (n, 1))
    ref = R.score(l, S.temperatures(0.7, n), None, tokens, 0)
    with R.Arena() as D:
        lg, tok, lp, st = D.put(bits), D.put(tokens.astype(np.int32)), D.room(4 * n, 0xee), D.room(8 * n, 0xee)
        W = gpu.Workspace(gpu.lib().d3s_logprob_workspace_bytes(gpu.DTYPE_BF16, n, V, top))
        D.held.append(W.buf)
        assert gpu.logprob_raw(lg.ptr, gpu.DTYPE_BF16, n, V, V, 0.7, None, tok.ptr, 1, lp.ptr, None, st.ptr, top,
                               workspace=W.arg()) == 0
        hiprt.synchronize()
        R.assert_near(lp.download((n, 1), np.float32), ref["logprobs"], R.score_tol(ref, ref["logprobs"]))
        R.assert_near(st.download((n, 2), np.float32)[:, 0], ref["m"], 0)
