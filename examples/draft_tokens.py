#!/usr/bin/env python3
"""A small model drafts tokens, a larger one verifies several at once, and the small
one is tuned on what the larger one draws, on one GPU: the sampler's library does every
lookup, norm, product, draw, verification, score and gradient.

    python3 examples/draft_tokens.py [--steps N] [--seqs B] [--drafts L] [--vocab V] [--top-k K]

A model takes the last CONTEXT tokens of a sequence, each place with a part of the table
of its own:
  e = sum_t table[t, id_t]                     d3s_embed
  y = rmsnorm(e) gain                          d3s_rms_norm
  logits = y w^T                               d3s_dense_bf16
A round of decoding for all sequences:
  L times: the small model's logits and a draw  d3s_sample
  the large model's logits after each of them, in one batch
  the drafts accepted, and the next token       d3s_verify (whole rows), or with --top-k
                                                d3s_verify_ranked (the candidates that d3s_sample wrote)
A step of tuning the small model, on contexts and the tokens that followed them:
  e = dropout(sum_t table[t, id_t])            d3s_embed, d3s_dropout
  y, logits as above; log p of the tokens      d3s_logprob
  d logits, in place                           d3s_logprob_backward
  d y = d logits w, d w = d logits^T y         d3s_dense_bf16
  d e, d gain                                  d3s_rms_norm_backward
  the same dropout of d e                      d3s_dropout
  d table                                      d3s_embed_backward
  clipped, weights -= rate * gradients         d3s_clip_grads, torch
Random weights: the large model is a fixed random function."""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "drama3-mlx_amd"))
import d3s  # noqa: E402

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
CONTEXT, EPS = 4, 1e-6


def check(status, what):
    if status != d3s.OK:
        raise RuntimeError(f"{what}: status {status}")


def stream():
    return torch.cuda.current_stream().cuda_stream or None


def new(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def dense(x, w, y, x_transposed=False, w_transposed=False):
    m, n = y.shape
    k = x.shape[0] if x_transposed else x.shape[1]
    check(d3s.dense_raw(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), m, n, k, y.data_ptr(), y.stride(0),
                        d3s.DTYPE_F32 if y.dtype == F32 else d3s.DTYPE_BF16, x_transposed=x_transposed,
                        w_transposed=w_transposed, stream=stream()), "dense")


class Model:
    def __init__(self, vocab, width, spread, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.vocab, self.width = vocab, width
        self.master = {"table": normal(CONTEXT * vocab, width) * 0.2, "gain": 1 + 0.1 * normal(width),
                       "head": normal(vocab, width) * (spread * width ** -0.5)}
        self.master["table"][-vocab:] *= 5  # mostly the last token decides
        self.weights = {n: t.to(BF16) for n, t in self.master.items()}

    def embed(self, ids):
        rows, e = ids.shape[0], new(ids.shape[0], self.width)
        table = self.weights["table"]
        check(d3s.embed_raw(ids.data_ptr(), rows, CONTEXT, table.data_ptr(), d3s.DTYPE_BF16, self.width, self.vocab, self.vocab,
                            self.width, 1.0, e.data_ptr(), d3s.DTYPE_BF16, self.width, stream=stream()), "embed")
        return e

    def logits(self, e, rstd=None):
        """(logits [rows, vocab], the normed rows)"""
        rows, y = e.shape[0], new(*e.shape)
        check(d3s.rms_norm_raw(e.data_ptr(), d3s.DTYPE_BF16, self.width, None, 0, None, 0, self.weights["gain"].data_ptr(), EPS,
                               rows, self.width, y.data_ptr(), d3s.DTYPE_BF16, self.width,
                               rstd=None if rstd is None else rstd.data_ptr(), stream=stream()), "rms_norm")
        logits = new(rows, (self.vocab + 7) // 8 * 8)[:, :self.vocab]  # rows padded to whole 16 bytes
        dense(y, self.weights["head"], logits)
        return logits, y

    def __call__(self, ids):
        return self.logits(self.embed(ids))[0]


def sample(logits, u, top_p, cand=None, probs=None):
    rows, vocab = logits.shape
    ids = new(rows, dtype=I32)
    check(d3s.sample_raw(logits.data_ptr(), d3s.DTYPE_BF16, rows, vocab, logits.stride(0), u.data_ptr(), u.shape[1], 1.0, top_p,
                         None, ids.data_ptr(), None if probs is None else probs.data_ptr(),
                         None if cand is None else cand.data_ptr(), stream=stream()), "sample")
    return ids


def decode(target, small, history, drafts, top_k=0, top_p=0.9, seen=None):
    """One round: history [seqs, >= CONTEXT] int32; (tokens [seqs, drafts + 1], accepted [seqs]).
    top_k 0: draws from the whole rows; seen: a list that receives what was verified"""
    n, vocab = history.shape[0], target.vocab
    k = min(top_k, vocab) or vocab
    ranked = top_k > 0
    uniform = lambda *s: torch.randint(0, 1 << 24, s, device="cuda").float() * 2.0 ** -24  # noqa: E731
    ctx, rows, cand, probs = history, [], [], []
    for _ in range(drafts):
        logits = small(ctx[:, -CONTEXT:].contiguous())
        c, p = (new(n, k, dtype=I32), new(n, k, dtype=F32)) if ranked else (None, None)
        ids = sample(logits, uniform(n, k), top_p if ranked else 1.0, c, p)
        ctx = torch.cat([ctx, ids[:, None]], 1)
        rows.append(logits), cand.append(c), probs.append(p)
    drafted = ctx[:, -drafts:].contiguous()
    # the contexts after 0 .. drafts of the drafts, sequence by sequence
    after = ctx[:, -(drafts + CONTEXT):].unfold(1, CONTEXT, 1).contiguous()
    logits = target(after.view(-1, CONTEXT))
    tokens, accepted = new(n, drafts + 1, dtype=I32), new(n, dtype=I32)
    u = uniform(n, drafts)
    if ranked:
        tc, tp = new(n * (drafts + 1), k, dtype=I32), new(n * (drafts + 1), k, dtype=F32)
        sample(logits, uniform(n * (drafts + 1), k), top_p, tc, tp)
        dc, dp, ud = torch.stack(cand, 1), torch.stack(probs, 1), uniform(n, k)
        check(d3s.verify_ranked_raw(tc.data_ptr(), tp.data_ptr(), k, dc.data_ptr(), dp.data_ptr(), k, n, drafts,
                                    drafted.data_ptr(), None, u.data_ptr(), ud.data_ptr(), tokens.data_ptr(),
                                    accepted.data_ptr(), stream=stream()), "verify_ranked")
        what = dict(target_cand=tc, target_probs=tp, draft_cand=dc, draft_probs=dp)
    else:
        draft, ud = torch.stack(rows, 1), uniform(n)
        check(d3s.verify_raw(logits.data_ptr(), d3s.DTYPE_BF16, logits.stride(0), draft.data_ptr(), d3s.DTYPE_BF16,
                             draft.stride(1), n, drafts, vocab, drafted.data_ptr(), None, 1.0, 1.0, u.data_ptr(),
                             ud.data_ptr(), tokens.data_ptr(), accepted.data_ptr(), stream=stream()), "verify")
        what = dict(target=logits, draft=draft)
    if seen is not None:
        seen.append(dict(what, drafted=drafted, u_accept=u, u_draw=ud, tokens=tokens, accepted=accepted))
    return tokens, accepted


class Tuner:
    def __init__(self, model, rows, dropout=0.1, rate=4.0, max_norm=1.0, seed=5):
        self.model, self.rows, self.p, self.rate, self.max_norm, self.seed, self.count = model, rows, dropout, rate, max_norm, seed, 0
        self.grads = {n: torch.zeros_like(t) for n, t in model.master.items()}
        self.norm, self.rstd = new((), dtype=F32), new(rows, dtype=F32)
        self.logprobs, self.stats = new(rows, 1, dtype=F32), new(rows, 2, dtype=F32)
        self.grad_logprobs = torch.full((rows, 1), -1.0 / rows, device="cuda")
        names = list(self.grads)
        self.addresses = np.array([self.grads[n].data_ptr() for n in names], np.uint64)
        self.numel = np.array([self.grads[n].numel() for n in names], np.int64)
        self.dtypes = np.full(len(names), d3s.DTYPE_F32, np.int32)

    def dropout(self, x, draw):
        """in place"""
        check(d3s.dropout_raw(x.data_ptr(), d3s.DTYPE_BF16, x.stride(0), None, 0, x.shape[0], x.shape[1], self.p, self.seed, draw,
                              None, x.data_ptr(), x.stride(0), stream=stream()), "dropout")

    def gradients(self, ids, tokens):
        """the loss, -mean log p of tokens [rows] after contexts ids [rows, CONTEXT], and its gradients in self.grads"""
        m, g, draw = self.model, self.grads, self.count
        V, W = m.vocab, m.width
        e = m.embed(ids)
        self.dropout(e, draw)
        logits, y = m.logits(e, self.rstd)
        rows = (logits.data_ptr(), d3s.DTYPE_BF16, self.rows, V, logits.stride(0), 1.0, None, tokens.data_ptr(), 1)
        check(d3s.logprob_raw(*rows, self.logprobs.data_ptr(), None, self.stats.data_ptr(), stream=stream()), "logprob")
        check(d3s.logprob_backward_raw(*rows, self.stats.data_ptr(), None, self.grad_logprobs.data_ptr(), None, logits.data_ptr(),
                                       logits.stride(0), stream=stream()), "logprob_backward")
        dy = new(self.rows, W)
        dense(logits, m.weights["head"], dy, w_transposed=True)
        dense(logits, y, g["head"], x_transposed=True, w_transposed=True)
        check(d3s.rms_norm_backward_raw(dy.data_ptr(), d3s.DTYPE_BF16, W, e.data_ptr(), W, m.weights["gain"].data_ptr(),
                                        self.rstd.data_ptr(), None, 0, self.rows, W, dy.data_ptr(), W, g["gain"].data_ptr(),
                                        stream=stream()), "rms_norm_backward")
        self.dropout(dy, draw)
        check(d3s.embed_backward_raw(ids.data_ptr(), self.rows, CONTEXT, dy.data_ptr(), d3s.DTYPE_BF16, W, V, V, W, 1.0, False,
                                     g["table"].data_ptr(), d3s.DTYPE_F32, W, stream=stream()), "embed_backward")
        self.count += 1
        return -self.logprobs.mean()

    def step(self, ids, tokens):
        loss = self.gradients(ids, tokens)
        at = self.addresses.ctypes.data
        check(d3s.clip_grads_raw(at, at, self.numel.ctypes.data, self.dtypes.ctypes.data, len(self.numel), self.max_norm,
                                 self.norm.data_ptr(), stream=stream()), "clip_grads")
        for name, t in self.model.master.items():
            t.sub_(self.grads[name], alpha=self.rate)
            self.model.weights[name].copy_(t)
        return loss


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("steps", 200), ("seqs", 1024), ("drafts", 4), ("vocab", 64), ("top-k", 0)):
        p.add_argument("--" + name, type=int, default=value)
    a = p.parse_args(argv)
    target, small = Model(a.vocab, 512, 4.0, 1), Model(a.vocab, 128, 1.0, 2)
    tuner = Tuner(small, a.seqs)
    history = torch.randint(0, a.vocab, (a.seqs, CONTEXT), device="cuda").to(I32)
    shares = []
    for s in range(a.steps):
        tokens, accepted = decode(target, small, history, a.drafts, a.top_k)
        shares.append(float(accepted.float().mean()) / a.drafts)
        loss = tuner.step(history[:, -CONTEXT:].contiguous(), tokens[:, 0].contiguous())
        # (sequences keep one new token a round, so that all have one length)
        history = torch.cat([history, tokens[:, :1]], 1)[:, -CONTEXT:].contiguous()
        if s % 20 == 19:
            print(f"step {s}: loss {float(loss):.4f}, gradient norm {float(tuner.norm):.4f}, drafts accepted "
                  f"{sum(shares[-20:]) / 20:.3f}", flush=True)
    return shares


if __name__ == "__main__":
    main()
