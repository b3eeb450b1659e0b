#!/usr/bin/env python3
"""Tunes an adapter and a model's codebook heads on given codes, on one GPU: the
sampler's library does every product, draw, score and gradient.

    python3 examples/tune_heads.py [--steps N] [--rows R] [--width W] [--heads H] [--vocab V]

A step, for hidden states x [rows, width] of a frozen backbone and a code for each
row and head:
  h = x + silu(x a^T + b)                      d3s_dense_bf16 (the pre-activation kept)
  logits_i = h w_i^T                           d3s_dense_bf16
  the codes' log probabilities and entropies   d3s_logprob
  loss = -mean(log p) - 0.01 mean(entropy)
  d logits_i, in place                         d3s_logprob_backward
  d h += d logits_i w_i, d w_i = d logits_i^T h   d3s_dense_bf16, operands transposed
  d z = d h silu'(z), d b                      d3s_dense_activation_backward_bf16
  d a = d z^T x                                d3s_dense_bf16
  all gradients clipped to a norm of 1         d3s_clip_grads
  weights -= rate * gradients                  (fp32 copies, by torch)
and every few steps a draw from the heads with its log probability, as a server
would answer (d3s_sample, d3s_logprob).  Synthetic data: the codes are a fixed
random function of the states."""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "drama3-mlx_amd"))
import d3s  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
ENTROPY = 0.01


def check(status, what):
    if status != d3s.OK:
        raise RuntimeError(f"{what}: status {status}")


def stream():
    return torch.cuda.current_stream().cuda_stream or None


def dense(x, w, y, x_transposed=False, w_transposed=False, bias=None, act="none", residual=None, z=None):
    """y = residual + act(x w^T + bias), operands as stored"""
    m, n = y.shape
    k = x.shape[0] if x_transposed else x.shape[1]
    check(d3s.dense_raw(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), m, n, k, y.data_ptr(), y.stride(0),
                        d3s.DTYPE_F32 if y.dtype == F32 else d3s.DTYPE_BF16, x_transposed=x_transposed,
                        w_transposed=w_transposed, bias=None if bias is None else bias.data_ptr(),
                        activation=d3s.ACTIVATIONS[act], residual=None if residual is None else residual.data_ptr(),
                        residual_stride=0 if residual is None else residual.stride(0),
                        z=None if z is None else z.data_ptr(), z_stride=0 if z is None else z.stride(0),
                        stream=stream()), "dense")


class Tuner:
    def __init__(self, rows, width, heads, vocab, rate=0.5, max_norm=1.0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        new = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.rows, self.width, self.vocab, self.rate, self.max_norm = rows, width, vocab, rate, max_norm
        self.master = {"a": new(width, width) * (0.5 * width ** -0.5), "b": torch.zeros(width, device="cuda")}
        for i in range(heads):
            self.master[f"w{i}"] = new(vocab, width) * width ** -0.5
        self.heads = heads
        self.weights = {name: t.to(BF16) for name, t in self.master.items()}
        self.grads = {name: torch.zeros_like(t) for name, t in self.master.items()}
        e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.z, self.h, self.dh, self.dz = (e(rows, width) for _ in range(4))
        # rows of logits padded to whole 16 bytes
        self.logits = [e(rows, (vocab + 7) // 8 * 8)[:, :vocab] for _ in range(heads)]
        self.logprobs, self.entropy = e(heads, rows, 1, dtype=F32), e(heads, rows, dtype=F32)
        self.stats, self.norm = e(heads, rows, 2, dtype=F32), e((), dtype=F32)
        self.grad_logprobs = torch.full((rows, 1), -1.0 / (rows * heads), device="cuda")
        self.grad_entropy = torch.full((rows,), -ENTROPY / (rows * heads), device="cuda")
        names = list(self.grads)
        self.addresses = np.array([self.grads[n].data_ptr() for n in names], np.uint64)
        self.numel = np.array([self.grads[n].numel() for n in names], np.int64)
        self.dtypes = np.full(len(names), d3s.DTYPE_F32, np.int32)

    def forward(self, x):
        w = self.weights
        dense(x, w["a"], self.h, bias=w["b"], act="silu", residual=x, z=self.z)
        for i, logits in enumerate(self.logits):
            dense(self.h, w[f"w{i}"], logits)

    def _rows(self, i, codes):
        l = self.logits[i]  # noqa: E741
        return l.data_ptr(), d3s.DTYPE_BF16, self.rows, self.vocab, l.stride(0), 1.0, None, codes.data_ptr(), 1

    def score(self, codes):
        for i in range(self.heads):
            check(d3s.logprob_raw(*self._rows(i, codes[i]), self.logprobs[i].data_ptr(), self.entropy[i].data_ptr(),
                                  self.stats[i].data_ptr(), stream=stream()), "logprob")

    def backward(self, x, codes):
        w, g = self.weights, self.grads
        for i, dl in enumerate(self.logits):
            check(d3s.logprob_backward_raw(*self._rows(i, codes[i]), self.stats[i].data_ptr(),
                                           self.entropy[i].data_ptr(), self.grad_logprobs.data_ptr(),
                                           self.grad_entropy.data_ptr(), dl.data_ptr(), dl.stride(0),
                                           stream=stream()), "logprob_backward")
            dense(dl, w[f"w{i}"], self.dh, w_transposed=True, residual=self.dh if i else None)
            dense(dl, self.h, g[f"w{i}"], x_transposed=True, w_transposed=True)
        check(d3s.dense_activation_backward_raw(self.dh.data_ptr(), self.width, self.z.data_ptr(), self.width, self.rows,
                                                self.width, d3s.ACTIVATIONS["silu"], self.dz.data_ptr(), self.width,
                                                g["b"].data_ptr(), stream=stream()), "dense_activation_backward")
        dense(self.dz, x, g["a"], x_transposed=True, w_transposed=True)

    def step(self, x, codes):
        """one step on x [rows, width] bf16 and codes [heads, rows] int32: the loss before it"""
        self.forward(x)
        self.score(codes)
        loss = -self.logprobs.mean() - ENTROPY * self.entropy.mean()
        self.backward(x, codes)
        at = self.addresses.ctypes.data
        check(d3s.clip_grads_raw(at, at, self.numel.ctypes.data, self.dtypes.ctypes.data, len(self.numel), self.max_norm,
                                 self.norm.data_ptr(), stream=stream()), "clip_grads")
        for name, t in self.master.items():
            t.sub_(self.grads[name], alpha=self.rate)
            self.weights[name].copy_(t)
        return loss

    def draw(self, x, top_k=30, top_p=0.9):
        """codes [heads, rows] drawn from the heads, and their log probabilities"""
        self.forward(x)
        codes = torch.empty(self.heads, self.rows, dtype=torch.int32, device="cuda")
        k = min(top_k, self.vocab)
        for i, l in enumerate(self.logits):  # noqa: E741
            u = torch.rand(self.rows, k, device="cuda")
            check(d3s.sample_raw(l.data_ptr(), d3s.DTYPE_BF16, self.rows, self.vocab, l.stride(0), u.data_ptr(), k, 1.0,
                                 top_p, None, codes[i].data_ptr(), stream=stream()), "sample")
        self.score(codes)
        return codes, self.logprobs[:, :, 0]


def data(rows, width, heads, vocab, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, width, device="cuda", generator=g)
    codes = torch.stack([(x @ torch.randn(width, vocab, device="cuda", generator=g)).argmax(1) for _ in range(heads)])
    return x.to(BF16), codes.to(torch.int32)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("steps", 20), ("rows", 1024), ("width", 2048), ("heads", 10), ("vocab", 4097)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    tuner = Tuner(a.rows, a.width, a.heads, a.vocab)
    x, codes = data(a.rows, a.width, a.heads, a.vocab)
    losses = []
    for s in range(a.steps):
        losses.append(float(tuner.step(x, codes)))
        print(f"step {s}: loss {losses[-1]:.4f}, gradient norm {float(tuner.norm):.4f}", flush=True)
        if s % 10 == 9:
            drawn, logprobs = tuner.draw(x)
            print(f"  drawn codes that are the given ones: {float((drawn == codes).float().mean()):.3f}, "
                  f"their mean log probability {float(logprobs.mean()):.3f}", flush=True)
    return losses


if __name__ == "__main__":
    main()
