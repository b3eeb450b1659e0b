"""The example that tunes heads: its loss falls, and one step's gradients are the
loss's, by torch's own differentiation in 64 bits on the CPU.  It runs in a process
of its own, since torch brings its own HIP runtime."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.gpu
def test_tune_heads():
    import hiprt
    if hiprt.device_count() < 1:
        pytest.skip("no GPU")
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], cwd=HERE, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-4000:])
    assert r.stdout.strip().endswith("all checked")


def loss_falls(example):
    losses = example.main(["--steps", "12", "--rows", "300", "--width", "256", "--heads", "3", "--vocab", "1025"])
    assert all(b < a for a, b in zip(losses, losses[1:])) and losses[-1] < losses[0] - 0.05


def gradients(example):
    import torch
    rows, width, heads, vocab = 150, 200, 2, 333
    t = example.Tuner(rows, width, heads, vocab, max_norm=1e9)
    x, codes = example.data(rows, width, heads, vocab)
    w = {n: v.double().cpu().requires_grad_() for n, v in t.weights.items()}
    loss = t.step(x, codes)

    xd = x.double().cpu()
    h = xd + torch.nn.functional.silu(xd @ w["a"].t() + w["b"])
    total = 0.0
    for i in range(heads):
        logp = torch.log_softmax(h @ w[f"w{i}"].t(), 1)
        picked = logp.gather(1, codes[i].long().cpu()[:, None]).mean()
        total = total - (picked - example.ENTROPY * (logp.exp() * logp).sum(1).mean()) / heads
    total.backward()
    # z, h, the logits and the three kept gradients are rounded to bf16, each off by
    # at most 2^-8 of itself; a logit's error moves its probability by as much times
    # its size, which is below 5 here: ten such steps in all
    step = 2.0 ** -8
    assert abs(float(loss) - float(total)) < 5 * step
    for n, g in t.grads.items():
        ref = w[n].grad
        assert float((g.double().cpu() - ref).norm()) <= 10 * step * float(ref.norm()), n
    norm = sum(float(v.grad.square().sum()) for v in w.values()) ** 0.5
    assert abs(float(t.norm) - norm) <= 10 * step * norm


def draws_and_their_log_probabilities(example):
    import torch
    t = example.Tuner(64, 128, 2, 600)
    x, _ = example.data(64, 128, 2, 600)
    codes, logprobs = t.draw(x)
    for i in range(2):
        ref = torch.log_softmax(t.logits[i].double().cpu(), 1).gather(1, codes[i].long().cpu()[:, None])[:, 0]
        assert (codes[i] >= 0).all() and (codes[i] < 600).all()
        # fp32 sums of 600 terms and the logarithm: fewer than 200 steps of 2^-24 of values below 16
        assert float((logprobs[i].double().cpu() - ref).abs().max()) < 200 * 16 * 2.0 ** -24


if __name__ == "__main__":
    sys.path.insert(0, os.path.join(HERE, "..", "examples"))
    import tune_heads
    for f in (loss_falls, gradients, draws_and_their_log_probabilities):
        print(f.__name__, flush=True)
        f(tune_heads)
    print("all checked")
