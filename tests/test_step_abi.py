"""The entry points between ids and logits refuse what they cannot take before anything
is launched (no GPU needed: no pointer below is looked at)."""
import ctypes
import math

import pytest

P = 4096  # an aligned address that is never read
Q, S = 2 * P, 3 * P


@pytest.fixture(scope="module")
def d3s():
    import d3s
    d3s.lib()
    return d3s


VERIFY = dict(target=P, target_dtype=1, target_stride=100, draft=P, draft_dtype=0, draft_stride=100, n_seqs=3, n_draft=4,
              vocab=100, drafted=P, lengths=None, temperature=1.0, draft_temperature=1.0, u_accept=P, u_draw=P, tokens=P,
              n_accepted=P)


@pytest.mark.parametrize("change,status", [
    (dict(target_dtype=2), -4), (dict(draft_dtype=7), -4), (dict(n_seqs=-1), -1), (dict(n_seqs=1 << 30), -1),
    (dict(n_draft=-1), -1), (dict(n_draft=65), -1), (dict(vocab=0), -1),
    (dict(vocab=1 << 24, target_stride=1 << 24, draft_stride=1 << 24), -2), (dict(target_stride=99), -1),
    (dict(draft_stride=99), -1), (dict(target_stride=1 << 41), -1), (dict(target=None), -1), (dict(target=P + 1), -1),
    (dict(draft=P + 2), -1), (dict(drafted=None), -1), (dict(u_accept=None), -1), (dict(u_draw=None), -1),
    (dict(tokens=None), -1), (dict(n_accepted=None), -1), (dict(n_seqs=0, target=None), 0)])
def test_verify(d3s, change, status):
    assert d3s.verify_raw(**{**VERIFY, **change}) == status
    if status not in (0, -1) or "stride" in str(change) or "n_" in str(change) or "vocab" in str(change):
        p = d3s.verify_params(**{**VERIFY, **change})
        want = status if status < 0 and "n_accepted" not in change else None
        got = d3s.lib().d3s_verify_workspace_bytes(ctypes.byref(p))
        assert got == want if want is not None else got >= 0


def test_verify_null(d3s):
    assert d3s.lib().d3s_verify(None, None) == -1
    assert d3s.lib().d3s_verify_workspace_bytes(None) == -1


def test_verify_workspace(d3s):
    big = dict(VERIFY, vocab=151936, target_stride=151936, draft_stride=151936, n_seqs=64)
    need = d3s.lib().d3s_verify_workspace_bytes(ctypes.byref(d3s.verify_params(**big)))
    assert need >= 0
    if need:
        assert d3s.verify_raw(**big, workspace=(P, need - 1)) == -7
        assert d3s.verify_raw(**big, workspace=(None, need)) == -7
        assert d3s.verify_raw(**big, workspace=(P + 4, need)) == -1
    assert d3s.verify_raw(**big, workspace=(P, -1)) == -1


RANKED = dict(target_cand=P, target_probs=P, target_k=30, draft_cand=P, draft_probs=P, draft_k=30, n_seqs=3, n_draft=4,
              drafted=P, lengths=None, u_accept=P, u_draw=P, tokens=P, n_accepted=P)


@pytest.mark.parametrize("change,status", [
    (dict(n_seqs=-1), -1), (dict(n_seqs=1 << 30), -1), (dict(n_draft=-1), -1), (dict(n_draft=65), -1),
    (dict(target_k=0), -1), (dict(draft_k=0), -1), (dict(target_k=1025), -2), (dict(draft_k=1025), -2),
    (dict(target_cand=None), -1), (dict(target_probs=None), -1), (dict(draft_cand=None), -1), (dict(draft_probs=None), -1),
    (dict(drafted=None), -1), (dict(u_accept=None), -1), (dict(u_draw=None), -1), (dict(tokens=None), -1),
    (dict(n_accepted=None), -1), (dict(n_seqs=0, tokens=None), 0)])
def test_verify_ranked(d3s, change, status):
    assert d3s.verify_ranked_raw(**{**RANKED, **change}) == status


EMBED = dict(ids=P, n_rows=5, n_ids=2, table=P, dtype=1, table_stride=64, vocab=10, slot_rows=0, width=64, scale=1.0, y=P,
             y_dtype=0, y_stride=64)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(y_dtype=2), -4), (dict(n_rows=-1), -1), (dict(n_rows=1 << 31), -1), (dict(n_ids=0), -1),
    (dict(n_ids=65), -1), (dict(vocab=0), -1), (dict(vocab=1 << 31), -1), (dict(slot_rows=-1), -1), (dict(width=-1), -1),
    (dict(table_stride=63), -1), (dict(y_stride=63), -1), (dict(ids=None), -1), (dict(ids=P + 2), -1), (dict(table=None), -1),
    (dict(table=P + 1), -1), (dict(y=None), -1), (dict(y=P + 2), -1), (dict(n_rows=0, ids=None, y=None), 0),
    (dict(width=0), 0)])
def test_embed(d3s, change, status):
    assert d3s.embed_raw(**{**EMBED, **change}) == status


GRAD = dict(ids=P, n_rows=5, n_ids=2, dy=P, dtype=1, dy_stride=64, vocab=10, slot_rows=10, width=64, scale=1.0,
            accumulate=0, grad=Q, grad_dtype=0, grad_stride=64)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(grad_dtype=2), -4), (dict(n_rows=-1), -1), (dict(n_rows=1 << 31), -1), (dict(n_ids=0), -1),
    (dict(n_ids=65), -1), (dict(vocab=0), -1), (dict(slot_rows=9), -1), (dict(slot_rows=-1), -1), (dict(width=-1), -1),
    (dict(dy_stride=63), -1), (dict(grad_stride=63), -1), (dict(ids=None), -1), (dict(dy=None), -1), (dict(dy=P + 1), -1),
    (dict(grad=None), -1), (dict(grad=P + 2), -1), (dict(width=0, grad=None), 0), (dict(n_rows=0, accumulate=1), 0)])
def test_embed_backward(d3s, change, status):
    assert d3s.embed_backward_raw(**{**GRAD, **change}) == status


def test_embed_backward_workspace(d3s):
    size = d3s.lib().d3s_embed_backward_workspace_bytes
    assert size(-1, 1, 10, 0, 8) == -1 and size(5, 0, 10, 0, 8) == -1 and size(5, 2, 10, 9, 8) == -1
    need = size(100000, 1, 151936, 0, 2048)
    assert need >= 0
    big = dict(GRAD, n_rows=100000, n_ids=1, vocab=151936, slot_rows=0, dy_stride=2048, width=2048, grad_stride=2048)
    if need:
        assert d3s.embed_backward_raw(**big, workspace=(P, need - 1)) == -7
        assert d3s.embed_backward_raw(**big, workspace=(P + 4, need)) == -1
    assert d3s.embed_backward_raw(**big, workspace=(P, -1)) == -1


NORM = dict(x=P, dtype=1, x_stride=64, residual=Q, residual_stride=64, sum=S, sum_stride=64, gain=P, eps=1e-6, n_rows=5,
            width=64, y=4 * P, y_dtype=1, y_stride=64, rstd=P)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(y_dtype=3), -4), (dict(n_rows=-1), -1), (dict(width=-1), -1), (dict(eps=-1.0), -1),
    (dict(eps=math.nan), -1), (dict(x_stride=63), -1), (dict(residual_stride=63), -1), (dict(sum_stride=63), -1),
    (dict(y_stride=63), -1), (dict(x=None), -1), (dict(x=P + 1), -1), (dict(y=None), -1), (dict(y=4 * P + 1), -1),
    (dict(gain=P + 1), -1), (dict(rstd=P + 2), -1), (dict(y=S), -1), (dict(y=P, y_dtype=0), -1),
    (dict(y=P, y_stride=80), -1), (dict(sum=Q, sum_stride=80), -1), (dict(sum=P, sum_stride=80), -1),
    (dict(y_dtype=2), -1), (dict(y_dtype=2, scales=P, group=16), -1), (dict(y_dtype=2, scales=P, group=512), -1),
    (dict(y_dtype=2, scales=P + 2, group=32), -1), (dict(y_dtype=2, scales=P, y=P), -1), (dict(n_rows=0, x=None), 0),
    (dict(width=0), 0)])
def test_rms_norm(d3s, change, status):
    assert d3s.rms_norm_raw(**{**NORM, **change}) == status


NORM_GRAD = dict(dy=P, dtype=1, dy_stride=64, h=Q, h_stride=64, gain=P, rstd=P, dsum=S, dsum_stride=64, n_rows=5, width=64,
                 dx=4 * P, dx_stride=64, dgain=P)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(n_rows=-1), -1), (dict(width=-1), -1), (dict(dy_stride=63), -1), (dict(h_stride=63), -1),
    (dict(dsum_stride=63), -1), (dict(dx_stride=63), -1), (dict(dy=None), -1), (dict(h=None), -1), (dict(rstd=None), -1),
    (dict(dy=P + 1), -1), (dict(h=P + 1), -1), (dict(gain=P + 1), -1), (dict(dx=P + 1), -1), (dict(dgain=P + 2), -1),
    (dict(dsum=S + 1), -1), (dict(dx=P, dx_stride=80), -1), (dict(dx=Q, dx_stride=80), -1), (dict(dx=S, dx_stride=80), -1),
    (dict(width=0), 0), (dict(dx=None, dgain=None), 0), (dict(n_rows=0, dgain=None), 0)])
def test_rms_norm_backward(d3s, change, status):
    assert d3s.rms_norm_backward_raw(**{**NORM_GRAD, **change}) == status


def test_rms_norm_backward_workspace(d3s):
    size = d3s.lib().d3s_rms_norm_backward_workspace_bytes
    assert size(-1, 10, 1) == -1 and size(10, -1, 1) == -1 and size(1000, 100, 0) == 0
    need = size(8192, 2048, 1)
    big = dict(NORM_GRAD, n_rows=8192, width=2048, dy_stride=2048, h_stride=2048, dsum_stride=2048, dx_stride=2048)
    assert need >= 0
    if need:
        assert d3s.rms_norm_backward_raw(**big, workspace=(P, need - 1)) == -7
        assert d3s.rms_norm_backward_raw(**big, workspace=(P + 4, need)) == -1
    assert d3s.rms_norm_backward_raw(**big, workspace=(P, -1)) == -1


DROP = dict(x=P, dtype=1, x_stride=64, residual=Q, residual_stride=64, n_rows=5, width=64, p=0.1, seed=1, draw=2,
            draw_add=None, y=S, y_stride=64)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -4), (dict(n_rows=-1), -1), (dict(width=-1), -1), (dict(p=-0.1), -1), (dict(p=1.1), -1),
    (dict(p=math.nan), -1), (dict(x_stride=63), -1), (dict(y_stride=63), -1), (dict(residual_stride=63), -1),
    (dict(x=None), -1), (dict(y=None), -1), (dict(x=P + 1), -1), (dict(y=S + 1), -1), (dict(residual=Q + 1), -1),
    (dict(draw_add=P + 4), -1), (dict(y=P, y_stride=80), -1), (dict(y=Q, y_stride=80), -1), (dict(n_rows=0, x=None), 0),
    (dict(width=0), 0)])
def test_dropout(d3s, change, status):
    assert d3s.dropout_raw(**{**DROP, **change}) == status


@pytest.mark.parametrize("slot_rows,status", [(0, 0), (9, -1), (10, 0), (25, 0)])
def test_parts_overlap_nowhere(d3s, slot_rows, status):
    """the lookup and its gradient take the same parts of a table (n_rows 0: nothing is launched)"""
    assert d3s.embed_raw(**{**EMBED, "n_rows": 0, "slot_rows": slot_rows}) == status
    need = d3s.lib().d3s_embed_backward_workspace_bytes(5, 2, 10, slot_rows, 64)
    assert need == -1 if status else need > 0


@pytest.mark.parametrize("n_rows,n_ids,fits", [((1 << 31) - 65536, 1, True), ((1 << 31) - 65535, 1, False),
                                               ((1 << 25) - 1024, 64, True), ((1 << 25) - 1023, 64, False)])
def test_ids_of_a_gradient(d3s, n_rows, n_ids, fits):
    need = d3s.lib().d3s_embed_backward_workspace_bytes(n_rows, n_ids, 10, 0, 8)
    assert need > 4 * n_rows * n_ids if fits else need == -1
    if not fits:
        assert d3s.embed_backward_raw(**{**GRAD, "n_rows": n_rows, "n_ids": n_ids, "slot_rows": 0}) == -1


@pytest.mark.parametrize("name", ["drafted", "lengths", "u_accept", "u_draw", "tokens", "n_accepted", "accept", "counters"])
def test_verification_between_words(d3s, name):
    """arrays of 32-bit words that begin between two"""
    assert d3s.verify_raw(**{**VERIFY, name: P + 2}) == -1
    assert d3s.verify_ranked_raw(**{**RANKED, name: P + 2}) == -1


@pytest.mark.parametrize("name", ["target_cand", "target_probs", "draft_cand", "draft_probs"])
def test_candidates_between_words(d3s, name):
    assert d3s.verify_ranked_raw(**{**RANKED, name: P + 2}) == -1


def test_room_for_the_chunks_of_a_gradient(d3s):
    """a million ids: rows of more than 32 are cut into chunks of 64 or more positions, at most two for 65, each of which
    has a row of sums"""
    size = d3s.lib().d3s_embed_backward_workspace_bytes
    n, chunks = 1000000, 2 * 1000000 // 65 + 1
    narrow, wide = size(n, 1, 5000, 0, 8), size(n, 1, 5000, 0, 4096)
    assert 0 < wide - narrow <= 4 * (4096 - 8) * chunks + 512
