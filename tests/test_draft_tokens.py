"""The example that drafts, verifies and tunes: it runs, one step's gradients are the loss's, by
torch's own differentiation in 64 bits on the CPU, and each verified round is the plain
form's.  It runs in a process of its own, since torch brings its own HIP runtime."""
import os
import subprocess
import sys

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.gpu
def test_draft_tokens():
    import hiprt
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], cwd=HERE, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-4000:])
    assert r.stdout.strip().endswith("all checked")


def runs(example):
    for more in ([], ["--top-k", "30"]):
        shares = example.main(["--steps", "10", "--seqs", "33", "--vocab", "301", "--drafts", "3"] + more)
        assert len(shares) == 10 and all(0 <= s <= 1 for s in shares)


def gradients(example):
    import torch
    import step_ref as SR
    rows, vocab, width = 150, 203, 96
    m = example.Model(vocab, width, 2.0, 3)
    t = example.Tuner(m, rows, dropout=0.3)
    g = torch.Generator(device="cuda").manual_seed(4)
    ids = torch.randint(0, vocab, (rows, example.CONTEXT), device="cuda", generator=g).to(torch.int32)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g).to(torch.int32)
    loss = t.gradients(ids, tokens)

    w = {n: v.double().cpu().requires_grad_() for n, v in m.weights.items()}
    at = ids.long().cpu() + torch.arange(example.CONTEXT) * vocab
    kept = torch.from_numpy(SR.uniforms(rows * width, t.seed, 0).reshape(rows, width) >= np.float32(t.p))
    e = w["table"][at].sum(1) * kept / (1 - float(np.float32(t.p)))
    y = e / (e.square().mean(1, keepdim=True) + example.EPS).sqrt() * w["gain"]
    logp = torch.log_softmax(y @ w["head"].t(), 1)
    total = -logp.gather(1, tokens.long().cpu()[:, None]).mean()
    total.backward()
    # e (twice), y, the logits, their gradient, dy, de and its dropout are rounded to bf16, each off
    # by at most 2^-8 of itself, a logit's error moving its probability by its size (below 8 here): 20 such steps
    step = 2.0 ** -8
    assert abs(float(loss) - float(total.detach())) < 20 * step
    for n, v in t.grads.items():
        ref = w[n].grad
        assert float((v.double().cpu() - ref).norm()) <= 20 * step * float(ref.norm()), n
    # rows of the table that no context names
    named = torch.zeros(len(w["table"]), dtype=torch.bool)
    named[at.flatten()] = True
    assert (t.grads["table"].cpu()[~named] == 0).all()


def verified_rounds(example):
    import torch
    import step_ref as SR
    import test_verify as TV
    n, L, vocab = 40, 4, 150
    target, small = example.Model(vocab, 128, 2.0, 6), example.Model(vocab, 64, 1.0, 7)
    torch.manual_seed(8)
    history = torch.randint(0, vocab, (n, example.CONTEXT), device="cuda").to(torch.int32)
    host = lambda v: v.float().cpu().numpy().astype(np.float64) if v.is_floating_point() else v.cpu().numpy()  # noqa: E731
    accepted = 0
    for top_k in (0, 0, 30, 30):
        seen = []
        tokens, _ = example.decode(target, small, history, L, top_k, seen=seen)
        s = {k: host(v) for k, v in seen[0].items()}
        if top_k:
            ref = TV.ranked_ref(s["target_cand"], s["target_probs"], s["draft_cand"], s["draft_probs"], s["drafted"], None,
                                s["u_accept"], s["u_draw"])
        else:
            one = np.ones(n)
            t = s["target"].reshape(n, L + 1, vocab)
            # (no draw of these lies where rounding decides)
            assert np.array_equal(SR.keep_off_borders(t, s["draft"], s["drafted"], one, one, s["u_accept"]), s["u_accept"])
            ref = SR.verify(t, s["draft"], s["drafted"], None, one, one, s["u_accept"], s["u_draw"])
        assert np.array_equal(s["tokens"], ref[0]) and np.array_equal(s["accepted"], ref[1]), top_k
        accepted += int(s["accepted"].sum())
        history = torch.cat([history, tokens[:, :1]], 1)[:, 1:].contiguous()
    assert accepted > 0


if __name__ == "__main__":
    for p in ("examples", "drama3-mlx_amd"):
        sys.path.insert(0, os.path.join(HERE, "..", p))
    sys.path.insert(0, HERE)
    import draft_tokens
    for f in (runs, gradients, verified_rounds):
        print(f.__name__, flush=True)
        f(draft_tokens)
    print("all checked")
