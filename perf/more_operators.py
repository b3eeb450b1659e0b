"""The operators between ids and logits as their callers issue them, for timing:
verification of drafted tokens (from whole rows of logits, and from the ranked
candidates of a filtered draw), embedding lookup and its gradient,
root-mean-square norm with the residual's addition (also with an output in 8
bits) and its gradient, and dropout whose mask is drawn again by its backward.

A case is a dict of plain values:
  kind     "verify" (d3s_verify), "verify_ranked" (d3s_verify_ranked),
           "embed" (d3s_embed), "embed_grad" (d3s_embed_backward),
           "norm" (d3s_rms_norm), "norm_grad" (d3s_rms_norm_backward) or
           "dropout" (d3s_dropout)
  seqs, drafts, vocab, dtype   sequences, drafted tokens of each, the logits;
           ragged: some sequences have fewer drafts; per_seq: a temperature for
           each; certain: the drafts come without probabilities; k: candidates
  rows, ids, width   ids looked up and summed for a row; slots: each of them has
           a part of the table of its own; zipf: frequent tokens, as text has
  out      the output's type; "e4m3": 8 bits, with an fp32 scale for each `group`
           elements of a row (0: one a row)
  residual, keep     a residual is added, and the sum written
  p        the probability that dropout drops an element
  pad      elements between two rows of the inputs

The widths 2048, 4096, 4097 and 151936, and 30 candidates, are those of
d3s_workloads.py and bench.py, the others generic.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

MIN_T = 1e-5
E4M3_MOST = 448.0
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}


def _d3s():
    if "d3s" not in sys.modules:
        sys.path.insert(0, os.path.abspath("drama3-mlx_amd"))
    import d3s
    return d3s


def _verify(name, seqs, drafts, vocab, dtype, ragged, per_seq, certain=False, pad=0):
    return dict(name=name, kind="verify", seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype, ragged=ragged,
                per_seq=per_seq, certain=certain, pad=pad)


def _ranked(name, seqs, drafts, k, draft_k, ragged):
    return dict(name=name, kind="verify_ranked", seqs=seqs, drafts=drafts, vocab=4097, k=k, draft_k=draft_k, ragged=ragged)


def _embed(name, kind, rows, ids, vocab, width, slots, dtype, out, zipf=False, pad=0):
    return dict(name=name, kind=kind, rows=rows, ids=ids, vocab=vocab, width=width, slots=slots, dtype=dtype, out=out,
                zipf=zipf, pad=pad)


def _norm(name, kind, rows, width, dtype, out, residual, keep, group=0, pad=0):
    return dict(name=name, kind=kind, rows=rows, width=width, dtype=dtype, out=out, residual=residual, keep=keep,
                group=group, pad=pad)


def _dropout(name, rows, width, dtype, residual, p, pad=0):
    return dict(name=name, kind="dropout", rows=rows, width=width, dtype=dtype, residual=residual, p=p, pad=pad)


def listed():
    return [
        # one stream's next four main tokens, drafted by a smaller model, checked at once
        _verify("verify_stream", 1, 4, 4097, "bf16", False, False),
        # a serving step over a text vocabulary: four drafts a request, fewer for some
        _verify("verify_text", 64, 4, 151936, "bf16", True, True),
        # the same step where both models draw among their thirty best candidates
        _ranked("verify_ranked", 64, 4, 30, 30, True),
        # a decoded frame's ten codes become the next step's input row
        _embed("embed_frame", "embed", 1, 10, 4097, 2048, True, "bf16", "bf16"),
        # a batch of prompts in text tokens
        _embed("embed_prompt", "embed", 8192, 1, 151936, 2048, False, "bf16", "bf16", zipf=True),
        # the codebooks' gradient of a batch of frames, ten codes each
        _embed("embed_grad_codes", "embed_grad", 4096, 10, 4097, 2048, True, "bf16", "f32"),
        # a text table's gradient: a few tokens very often, most of them never
        _embed("embed_grad_text", "embed_grad", 16384, 1, 151936, 1024, False, "bf16", "bf16", zipf=True),
        # the norm before the heads, one stream's next token
        _norm("norm_token", "norm", 1, 2048, "bf16", "bf16", True, True),
        # the same over a batch of prompts, for a product in 8 bits
        _norm("norm_prompt_e4m3", "norm", 8192, 2048, "bf16", "e4m3", True, True, group=128),
        # its gradient, with the residual path's
        _norm("norm_grad", "norm_grad", 8192, 2048, "bf16", "bf16", True, True),
        # a layer's output, dropped out before it joins the residual
        _dropout("dropout_prompt", 8192, 2048, "bf16", True, 0.1),
        # the backward of dropout over fp32 gradients of odd rows
        _dropout("dropout_grad_odd", 1000, 4097, "f32", False, 0.5),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "verify_ranked", "embed", "embed", "embed_grad", "embed_grad", "norm", "norm",
                       "norm_grad", "dropout", "dropout"])
    pad = rng.choice([0, 0, 8, rng.randint(1, 15)])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "verify":
        vocab = rng.choice([4096, 4097, 151936, _log(rng, 2, 200000)])
        drafts = rng.randint(1, 8)
        seqs = _log(rng, 1, min(512, max(1, 64 * 9 * 151936 // (vocab * (2 * drafts + 1)))))
        return dict(kind=kind, seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype, ragged=rng.random() < 0.5,
                    per_seq=rng.random() < 0.5, certain=rng.random() < 0.25, pad=pad)
    if kind == "verify_ranked":
        return dict(kind=kind, seqs=_log(rng, 1, 1024), drafts=rng.randint(1, 8), vocab=4097,
                    k=rng.choice([30, rng.randint(1, 64), _log(rng, 1, 512)]), draft_k=rng.choice([30, rng.randint(1, 64)]),
                    ragged=rng.random() < 0.5)
    width = rng.choice([2048, 4096, 8 * _log(rng, 4, 1024), _log(rng, 16, 8192)])
    rows = _log(rng, 1, min(16384, 8192 * 2048 // width))
    if kind in ("embed", "embed_grad"):
        slots = rng.random() < 0.5
        ids = rng.choice([10, rng.randint(2, 16)]) if slots else rng.choice([1, 1, rng.randint(2, 4)])
        vocab = rng.choice([4097, _log(rng, 2, 8192)]) if slots else rng.choice([151936, _log(rng, 2, 200000)])
        vocab = max(2, min(vocab, 151936 * 1024 // (width * (ids if slots else 1))))
        rows = max(1, rows // (ids if slots else 1))
        return dict(kind=kind, rows=rows, ids=ids, vocab=vocab, width=width, slots=slots, dtype=dtype,
                    out=rng.choice(["bf16", "f32"]), zipf=not slots and rng.random() < 0.6, pad=pad)
    if kind == "norm":
        residual = rng.random() < 0.6
        out = rng.choice([dtype, dtype, "e4m3"])
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, out=out, residual=residual,
                    keep=residual and rng.random() < 0.8, group=rng.choice([0, 32, 128]) if out == "e4m3" else 0, pad=pad)
    if kind == "norm_grad":
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, out=dtype, residual=rng.random() < 0.6, keep=True,
                    group=0, pad=pad)
    return dict(kind=kind, rows=rows, width=width, dtype=dtype, residual=rng.random() < 0.5,
                p=rng.choice([0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)]), pad=pad)


def _rows(shape, pad, dtype, g, scale=1.0):
    """a matrix whose rows lie `pad` elements apart"""
    t = torch.empty(shape[0], shape[1] + pad, dtype=dtype, device="cuda").normal_(0, scale, generator=g)
    return t[:, :shape[1]]


def _new(shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda")


def _uniforms(shape, g):
    """multiples of 2^-24 in [0, 1), as the framework's generator makes them"""
    return torch.randint(0, 1 << 24, shape, device="cuda", generator=g).float() * 2.0 ** -24


def _lengths(case, g):
    n, most = case["seqs"], case["drafts"]
    if not case["ragged"]:
        return None
    short = torch.randint(0, most + 1, (n,), device="cuda", generator=g)
    return torch.where(torch.rand(n, device="cuda", generator=g) < 0.4, short, most).to(torch.int32)


def _pair_of_logits(n, drafts, vocab, g):
    """[n, drafts + 1, vocab] of a target, [n, drafts, vocab] of a draft model near it"""
    target = torch.empty(n, drafts + 1, vocab, device="cuda").normal_(0, 2.5, generator=g)
    at = torch.randint(0, vocab, (n, drafts + 1, min(8, vocab)), device="cuda", generator=g)
    target.scatter_add_(2, at, torch.rand(at.shape, device="cuda", generator=g) * 6 + 4)  # a few likely tokens
    draft = target[:, :drafts] + torch.empty(n, drafts, vocab, device="cuda").normal_(0, 0.7, generator=g)
    return target, draft


def _drawn(logits, g):
    """tokens drawn from softmax(logits), by the exponential race"""
    e = torch.rand(logits.shape, device="cuda", generator=g).clamp_min_(1e-7).log_().neg_().log_()
    return (logits - e).argmax(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    kind, bf, f32, i32 = case["kind"], torch.bfloat16, torch.float32, torch.int32
    if kind in ("verify", "verify_ranked"):
        n, L, V = case["seqs"], case["drafts"], case["vocab"]
        target, draft = _pair_of_logits(n, L, V, g)
        s["lengths"] = _lengths(case, g)
        s["u_accept"] = _uniforms((n, L), g)
        s["out"] = dict(tokens=_new((n, L + 1), i32), n_accepted=_new((n,), i32), accept=_new((n, L), f32))
        if kind == "verify":
            dt = DT[case["dtype"]]
            s["T"] = torch.rand(n, device="cuda", generator=g) * 0.7 + 0.5 if case["per_seq"] else None
            T = 1.0 if s["T"] is None else s["T"][:, None, None]
            s["drafted"] = _drawn(draft / T, g).to(i32)
            s["target"] = _new((n * (L + 1), V + case["pad"]), dt)[:, :V]
            s["target"].copy_(target.view(-1, V))
            s["draft"] = None
            if case["certain"]:  # a draft model that only gives its best token
                s["drafted"] = draft.argmax(-1).to(i32)
            else:
                s["draft"] = _new((n * L, V + case["pad"]), dt)[:, :V]
                s["draft"].copy_(draft.view(-1, V))
            s["u_draw"] = _uniforms((n,), g)
        else:
            # what a draw with top_k and top_p = 0.9 writes: ids by rank, probabilities, 0 past the cut
            for name, l, k in (("target", target, case["k"]), ("draft", draft, case["draft_k"])):  # noqa: E741
                top = torch.topk(torch.softmax(l.double(), 2), k, 2)
                before = top.values.cumsum(2) - top.values
                kept = top.values.masked_fill((before + top.values > 0.9) & (torch.arange(k, device="cuda") > 0), 0)
                s[name + "_cand"] = top.indices.to(i32).contiguous()
                s[name + "_probs"] = (kept / kept.sum(2, keepdim=True)).float().contiguous()
            rank = _drawn(s["draft_probs"].log(), g)
            s["drafted"] = s["draft_cand"].gather(2, rank[:, :, None])[:, :, 0].contiguous()
            s["u_draw"] = _uniforms((n, case["k"]), g)
    elif kind in ("embed", "embed_grad"):
        R, t, V, W = case["rows"], case["ids"], case["vocab"], case["width"]
        if case["zipf"]:  # the token of rank r with a frequency of about 1 / r
            r = torch.exp(torch.rand(R, t, device="cuda", generator=g) * math.log(V + 1)) - 1
            ids = (r.long().clamp(0, V - 1) * 40503) % V
        else:
            ids = torch.randint(0, V, (R, t), device="cuda", generator=g)
        s["ids"] = torch.where(torch.rand(R, t, device="cuda", generator=g) < 0.02, -1, ids).to(i32)  # padding
        s["scale"] = W ** 0.5 if kind == "embed" and not case["slots"] else 1.0
        table_rows = V * t if case["slots"] else V
        if kind == "embed":
            s["table"] = _rows((table_rows, W), case["pad"], DT[case["dtype"]], g, W ** -0.5)
            s["out"] = dict(y=_new((R, W), DT[case["out"]]))
        else:
            s["dy"] = _rows((R, W), case["pad"], DT[case["dtype"]], g)
            s["out"] = dict(grad=_new((table_rows, W), DT[case["out"]]))
    else:
        R, W, pad, dt = case["rows"], case["width"], case["pad"], DT[case["dtype"]]
        s["x"] = _rows((R, W), pad, dt, g)
        s["residual"] = _rows((R, W), pad, dt, g, 2.0) if case["residual"] else None
        if kind == "dropout":
            s["seed"], s["draw"] = 0x9E3779B97F4A7C15 ^ seed, 2 * seed + 1
            s["out"] = dict(y=_new((R, W), dt))
            return s
        s["gain"] = (torch.empty(W, device="cuda").normal_(1, 0.2, generator=g)).to(dt)
        s["eps"] = 1e-6
        if kind == "norm":
            s["out"] = dict(y=_new((R, W), DT[case["out"]]), rstd=_new((R,), f32))
            if case["keep"]:
                s["out"]["sum"] = _new((R, W), dt)
            if case["out"] == "e4m3":
                s["out"]["scales"] = _new((R, -(-W // (case["group"] or W))), f32)
        else:
            # x is what the forward pass kept, residual the gradient that reaches it past the norm
            s["rstd"] = (s["x"].double().square().mean(1) + s["eps"]).rsqrt().float()
            s["dy"] = _rows((R, W), pad, dt, g)
            s["out"] = dict(dx=_new((R, W), dt), dgain=_new((W,), f32))
    return s


# ---- the plain forms: elementary operations in 32 bits ----
def _softmax(x, T):
    d = (x - x.amax(-1, keepdim=True)) / T
    e = d.exp()
    return e / e.sum(-1, keepdim=True)


def _logp_of(logits, tokens, T):
    """log softmax(logits / T) [n, l, V] at tokens [n, l], in 32 bits"""
    x = logits.float()
    top = x.amax(2, keepdim=True)
    d = (x - top) / T
    return d.gather(2, tokens[:, :, None].long())[:, :, 0] - d.exp().sum(2).log()


def _accepted(s, p, q):
    """(accepted in a row, the probability that each draft is accepted)"""
    n, L = p.shape
    place = torch.arange(L, device="cuda")
    there = place < s["lengths"][:, None] if s["lengths"] is not None else torch.ones(n, L, dtype=torch.bool, device="cuda")
    ok = there & (s["u_accept"] * q < p)
    accept = torch.where(q > 0, p / q, (p > 0).to(p.dtype)).clamp_max(1)
    return ok.long().cumprod(1).sum(1), torch.where(there, accept, 0.0), there


def _tokens(s, n_acc, token):
    """the accepted drafts, the drawn token, -1"""
    L = s["case"]["drafts"]
    place = torch.arange(L + 1, device="cuda")
    all_ = torch.cat([s["drafted"].long(), torch.zeros_like(n_acc)[:, None]], 1)
    out = torch.where(place < n_acc[:, None], all_, -1)
    return torch.where(place == n_acc[:, None], token[:, None], out).to(torch.int32)


def _plain_verify(s):
    case = s["case"]
    n, L, V = case["seqs"], case["drafts"], case["vocab"]
    T = torch.ones(n, device="cuda") if s["T"] is None else s["T"].clamp_min(MIN_T)
    target = s["target"].unflatten(0, (n, L + 1))
    p = _logp_of(target[:, :L], s["drafted"], T[:, None, None]).exp()
    if s["draft"] is None:
        q = torch.ones_like(p)
    else:
        draft = s["draft"].unflatten(0, (n, L))
        q = _logp_of(draft, s["drafted"], T[:, None, None]).exp()
    n_acc, accept, there = _accepted(s, p, q)
    # the drawn rows in 64 bits: their sums meet a border of u
    seq, i = torch.arange(n, device="cuda"), n_acc.clamp_max(L - 1)
    pr = _softmax(target[seq, n_acc].double(), T.double()[:, None])
    if s["draft"] is None:
        qr = torch.zeros_like(pr).scatter_(1, s["drafted"][seq, i].long()[:, None], 1)
    else:
        qr = _softmax(draft[seq, i].double(), T.double()[:, None])
    rejected = (n_acc < L) & there[seq, i]
    r = torch.where(rejected[:, None], (pr - qr).clamp_min(0), pr)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, pr)
    c = r.cumsum(1)
    token = (c <= s["u_draw"].double()[:, None] * c[:, -1:]).sum(1)
    last = torch.where(r > 0, torch.arange(V, device="cuda"), 0).amax(1)
    return dict(tokens=_tokens(s, n_acc, torch.minimum(token, last)), n_accepted=n_acc.to(torch.int32), accept=accept)


def _plain_ranked(s):
    case = s["case"]
    n, L = case["seqs"], case["drafts"]
    pc, pp, qc, qp = s["target_cand"], s["target_probs"], s["draft_cand"], s["draft_probs"]
    tok = s["drafted"][:, :, None]
    p = torch.where(pc[:, :L] == tok, pp[:, :L], 0.0).sum(2)
    q = torch.where(qc == tok, qp, 0.0).sum(2)
    n_acc, accept, there = _accepted(s, p, q)
    seq, i = torch.arange(n, device="cuda"), n_acc.clamp_max(L - 1)
    pr = pp[seq, n_acc]
    same = pc[seq, n_acc][:, :, None] == qc[seq, i][:, None, :]
    qr = torch.where(same, qp[seq, i][:, None, :], 0.0).sum(2)
    rejected = (n_acc < L) & there[seq, i]
    r = torch.where(rejected[:, None], (pr - qr).clamp_min(0), pr)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, pr)
    score = torch.where(r > 0, r / -torch.log(1 - s["u_draw"]), -1.0)
    token = pc[seq, n_acc].gather(1, score.argmax(1, keepdim=True))[:, 0]
    return dict(tokens=_tokens(s, n_acc, token.long()), n_accepted=n_acc.to(torch.int32), accept=accept)


def _table_rows(s):
    """(row of the table for each id, whether it is one)"""
    case, ids = s["case"], s["ids"].long()
    first = torch.arange(case["ids"], device="cuda") * (case["vocab"] if case["slots"] else 0)
    return ids.clamp_min(0) + first, (ids >= 0) & (ids < case["vocab"])


def _plain_embed(s):
    at, there = _table_rows(s)
    rows = s["table"][at].float() * there[:, :, None]
    return dict(y=(rows.sum(1) * s["scale"]).to(DT[s["case"]["out"]]))


def _plain_embed_grad(s):
    at, there = _table_rows(s)
    case, grad = s["case"], s["out"]["grad"]
    dy = s["dy"].float()[:, None, :].expand(-1, case["ids"], -1) * there[:, :, None]
    total = torch.zeros(grad.shape, device="cuda").index_add_(0, at.flatten(), dy.flatten(0, 1))
    return dict(grad=(total * s["scale"]).to(grad.dtype))


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    out = {}
    if s["residual"] is not None:
        x = x + s["residual"].float()
    if case["keep"]:
        out["sum"] = x.to(DT[case["dtype"]])
    rstd = 1 / (x.square().mean(1, keepdim=True) + s["eps"]).sqrt()
    y = x * rstd * s["gain"].float()
    out["rstd"] = rstd[:, 0]
    if case["out"] != "e4m3":
        out["y"] = y.to(DT[case["out"]])
        return out
    group = case["group"] or case["width"]
    y = torch.nn.functional.pad(y, (0, -case["width"] % group)).unflatten(1, (-1, group))
    scale = y.abs().amax(2) / E4M3_MOST
    q = (y / torch.where(scale > 0, scale, 1.0)[:, :, None]).clamp(-E4M3_MOST, E4M3_MOST)
    out["y"], out["scales"] = q.flatten(1)[:, :case["width"]].to(DT["e4m3"]), scale
    return out


def _plain_norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = s["x"].float() * rstd
    a = dy * s["gain"].float()
    dx = rstd * (a - xhat * (a * xhat).mean(1, keepdim=True))
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    return dict(dx=dx.to(s["x"].dtype), dgain=(dy * xhat).sum(0))


LOW = 0xFFFFFFFF


def _philox(quad, draw, seed):
    """the four words of each block of Philox4x32-10 (Salmon et al., SC'11), in int64"""
    c = [quad & LOW, (quad >> 32) & LOW, torch.full_like(quad, draw & LOW), torch.full_like(quad, (draw >> 32) & LOW)]
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # modulo 2^64: the halves are the product's
        c = [((b >> 32) & LOW) ^ c[1] ^ k0, b & LOW, ((a >> 32) & LOW) ^ c[3] ^ k1, a & LOW]
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack(c, 1)


def _plain_dropout(s):
    case, x = s["case"], s["x"].float()
    n = case["rows"] * case["width"]
    words = _philox(torch.arange(-(-n // 4), device="cuda"), s["draw"], s["seed"]).flatten()[:n].view(x.shape)
    u = (words >> 8).float() * 2.0 ** -24
    y = torch.where(u >= torch.tensor(case["p"], device="cuda"), x * (1 / (1 - case["p"])), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(s["x"].dtype))


# ---- the framework's calls ----
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    d3s, case, out = _d3s(), s["case"], s["out"]
    stream = torch.cuda.current_stream().cuda_stream or None
    kind = case["kind"]
    code = {"f32": d3s.DTYPE_F32, "bf16": d3s.DTYPE_BF16, "e4m3": d3s.DTYPE_E4M3}
    if kind == "verify":
        V, dt = case["vocab"], code[case["dtype"]]
        T = 1.0 if s["T"] is None else ("ptr", s["T"].data_ptr())
        rc = d3s.verify_raw(s["target"].data_ptr(), dt, s["target"].stride(0), _ptr(s["draft"]), dt, V + case["pad"],
                            case["seqs"], case["drafts"], V, s["drafted"].data_ptr(), _ptr(s["lengths"]), T, T,
                            s["u_accept"].data_ptr(), s["u_draw"].data_ptr(), out["tokens"].data_ptr(),
                            out["n_accepted"].data_ptr(), accept=out["accept"].data_ptr(), stream=stream)
    elif kind == "verify_ranked":
        rc = d3s.verify_ranked_raw(s["target_cand"].data_ptr(), s["target_probs"].data_ptr(), case["k"],
                                   s["draft_cand"].data_ptr(), s["draft_probs"].data_ptr(), case["draft_k"], case["seqs"],
                                   case["drafts"], s["drafted"].data_ptr(), _ptr(s["lengths"]), s["u_accept"].data_ptr(),
                                   s["u_draw"].data_ptr(), out["tokens"].data_ptr(), out["n_accepted"].data_ptr(),
                                   accept=out["accept"].data_ptr(), stream=stream)
    elif kind == "embed":
        rc = d3s.embed_raw(s["ids"].data_ptr(), case["rows"], case["ids"], s["table"].data_ptr(), code[case["dtype"]],
                           s["table"].stride(0), case["vocab"], case["vocab"] if case["slots"] else 0, case["width"],
                           s["scale"], out["y"].data_ptr(), code[case["out"]], case["width"], stream=stream)
    elif kind == "embed_grad":
        rc = d3s.embed_backward_raw(s["ids"].data_ptr(), case["rows"], case["ids"], s["dy"].data_ptr(),
                                    code[case["dtype"]], s["dy"].stride(0), case["vocab"],
                                    case["vocab"] if case["slots"] else 0, case["width"], s["scale"], False,
                                    out["grad"].data_ptr(), code[case["out"]], case["width"], stream=stream)
    elif kind == "norm":
        W = case["width"]
        rc = d3s.rms_norm_raw(s["x"].data_ptr(), code[case["dtype"]], s["x"].stride(0), _ptr(s["residual"]), W + case["pad"],
                              _ptr(out.get("sum")), W, s["gain"].data_ptr(), s["eps"], case["rows"], W, out["y"].data_ptr(),
                              code[case["out"]], W, group=case["group"], scales=_ptr(out.get("scales")),
                              rstd=out["rstd"].data_ptr(), stream=stream)
    elif kind == "norm_grad":
        W = case["width"]
        rc = d3s.rms_norm_backward_raw(s["dy"].data_ptr(), code[case["dtype"]], s["dy"].stride(0), s["x"].data_ptr(),
                                       s["x"].stride(0), s["gain"].data_ptr(), s["rstd"].data_ptr(), _ptr(s["residual"]),
                                       W + case["pad"], case["rows"], W, out["dx"].data_ptr(), W, out["dgain"].data_ptr(),
                                       stream=stream)
    else:
        W = case["width"]
        rc = d3s.dropout_raw(s["x"].data_ptr(), code[case["dtype"]], s["x"].stride(0), _ptr(s["residual"]),
                             W + case["pad"], case["rows"], W, case["p"], s["seed"], s["draw"], None, out["y"].data_ptr(),
                             W, stream=stream)
    if rc != d3s.OK:
        raise RuntimeError(f"{kind}: status {rc}")
    return out


def run(s):
    if own:
        return _own(s)
    return {"verify": _plain_verify, "verify_ranked": _plain_ranked, "embed": _plain_embed,
            "embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad,
            "dropout": _plain_dropout}[s["case"]["kind"]](s)


def work(case):
    kind = case["kind"]
    if kind == "verify":
        rows = case["seqs"] * (case["drafts"] + 1 + (0 if case["certain"] else case["drafts"]))
        return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + case["seqs"] * (16 * case["drafts"] + 12),
                "flops": 4 * rows * case["vocab"]}
    if kind == "verify_ranked":
        n, L = case["seqs"], case["drafts"]
        return {"bytes": n * (8 * ((L + 1) * case["k"] + L * case["draft_k"]) + 4 * case["k"] + 16 * L + 12),
                "flops": n * (2 * L * (case["k"] + case["draft_k"]) + 4 * case["k"])}
    if kind in ("embed", "embed_grad"):
        R, t, V, W = case["rows"], case["ids"], case["vocab"], case["width"]
        # rows of the table that some id names: of the codes' about all but e^(-ids / rows), of text's fewer
        table = V * t if case["slots"] else V
        named = min(R * t, table) if not case["zipf"] else min(R * t, table) / 2
        size, out = SIZE[case["dtype"]], SIZE[case["out"]]
        if kind == "embed":
            return {"bytes": 4 * R * t + named * W * size + R * W * out, "flops": R * t * W}
        return {"bytes": 4 * R * t + R * W * size + table * W * out, "flops": R * t * W}
    n, size = case["rows"] * case["width"], SIZE[case["dtype"]]
    if kind == "norm":
        scales = 4 * case["rows"] * -(-case["width"] // (case["group"] or case["width"])) if case["out"] == "e4m3" else 0
        return {"bytes": n * (size * (1 + case["residual"] + case["keep"]) + SIZE[case["out"]]) + scales +
                4 * case["rows"] + size * case["width"], "flops": 5 * n}
    if kind == "norm_grad":
        return {"bytes": n * size * (3 + case["residual"]) + 4 * case["rows"] + (4 + size) * case["width"], "flops": 9 * n}
    return {"bytes": n * size * (2 + case["residual"]), "flops": 2 * n}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "verify_ranked": _exact_verify, "embed": _exact_embed, "embed_grad": _exact_embed_grad,
            "norm": _exact_norm, "norm_grad": _exact_norm_grad, "dropout": _exact_dropout}[case["kind"]](s)


def _exact_verify(s):
    """a sequence and a place at a time, on probabilities over the whole vocabulary"""
    case = s["case"]
    n, L, V = case["seqs"], case["drafts"], case["vocab"]
    ranked = case["kind"] == "verify_ranked"

    def dist(name, seq, i):
        if ranked:
            p = torch.zeros(V, dtype=torch.float64, device="cuda")
            p[s[name + "_cand"][seq, i].long()] = s[name + "_probs"][seq, i].double()
            return p
        if s[name] is None:
            return torch.nn.functional.one_hot(s["drafted"][seq, i].long(), V).double()
        T = 1.0 if s["T"] is None else max(float(s["T"][seq]), MIN_T)
        return torch.softmax(s[name][seq * (L + (name == "target")) + i].double() / T, 0)

    accept = torch.zeros(n, L, dtype=torch.float64)
    for seq in range(n):
        for i in range(L if s["lengths"] is None else int(s["lengths"][seq])):
            x = int(s["drafted"][seq, i])
            p, q = float(dist("target", seq, i)[x]), float(dist("draft", seq, i)[x])
            accept[seq, i] = min(1.0, p / q)
    # the ids have to be the plain form's own
    return dict(accept=accept.cuda(), tokens=None, n_accepted=None)


def _exact_embed(s):
    case = s["case"]
    total = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
    for t in range(case["ids"]):
        ids = s["ids"][:, t].long()
        live = (ids >= 0).nonzero()[:, 0]
        total[live] += s["table"][ids[live] + t * case["vocab"] * case["slots"]].double()
    return dict(y=total * s["scale"])


def _exact_embed_grad(s):
    """each id's rows of dy, sorted by id and summed by differences of a running sum, a strip of columns at a time"""
    case = s["case"]
    ids = s["ids"].long() + torch.arange(case["ids"], device="cuda") * case["vocab"] * case["slots"]
    row = torch.arange(case["rows"], device="cuda")[:, None].expand_as(ids)
    keep = s["ids"] >= 0
    ids, order = ids[keep].sort()
    row = row[keep][order]
    out = torch.zeros(s["out"]["grad"].shape, dtype=torch.float64, device="cuda")
    named, count = ids.unique_consecutive(return_counts=True)
    end = count.cumsum(0)
    for c in range(0, case["width"], 256):
        run_ = torch.nn.functional.pad(s["dy"][:, c:c + 256].double()[row].cumsum(0), (0, 0, 1, 0))
        out[named, c:c + 256] = (run_[end] - run_[end - count]) * s["scale"]
    return dict(grad=out)


def _exact_norm(s):
    case = s["case"]
    h = s["x"].double() if s["residual"] is None else s["x"].double().add(s["residual"])
    rstd = torch.rsqrt((h * h).sum(1) / case["width"] + s["eps"])
    y = torch.einsum("rw,r,w->rw", h, rstd, s["gain"].double())
    out = dict(rstd=rstd, y=y)
    if case["keep"]:
        out["sum"] = h
    if case["out"] == "e4m3":
        width, group = case["width"], case["group"] or case["width"]
        scales = torch.stack([y[:, c:c + group].abs().max(1).values for c in range(0, width, group)], 1) / E4M3_MOST
        out["y"], out["scales"] = y / scales.repeat_interleave(group, 1)[:, :width], scales
    return out


def _exact_norm_grad(s):
    """torch's own differentiation of the norm with rstd's derivative written out"""
    h = s["x"].double().requires_grad_()
    gain = s["gain"].double().requires_grad_()
    rstd = s["rstd"].double()[:, None]
    mean = (h * h).mean(1, keepdim=True)
    # rstd as it was given, with the slope -rstd^3 / 2 in the mean square
    slope = rstd - 0.5 * rstd ** 3 * (mean - mean.detach())
    dx, dgain = torch.autograd.grad(h * slope * gain, (h, gain), s["dy"].double())
    return dict(dx=dx if s["residual"] is None else dx + s["residual"].double(), dgain=dgain)


def _exact_dropout(s):
    """Philox by numpy's unsigned integers"""
    case = s["case"]
    n = case["rows"] * case["width"]
    u32, u64 = np.uint32, np.uint64
    quad = np.arange(-(-n // 4), dtype=u64)
    half = lambda v: ((v & u64(LOW)).astype(u32), (v >> u64(32)).astype(u32))  # noqa: E731
    x0, x1 = half(quad)
    x2, x3 = (np.full_like(x0, (s["draw"] >> sh) & LOW) for sh in (0, 32))
    key = [s["seed"] & LOW, (s["seed"] >> 32) & LOW]
    for _ in range(10):
        lo0, hi0 = half(x0.astype(u64) * u64(0xD2511F53))
        lo1, hi1 = half(x2.astype(u64) * u64(0xCD9E8D57))
        x0, x1, x2, x3 = hi1 ^ x1 ^ u32(key[0]), lo1, hi0 ^ x3 ^ u32(key[1]), lo0
        key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
    words = np.stack([x0, x1, x2, x3], 1).reshape(-1)[:n].reshape(case["rows"], case["width"])
    kept = torch.from_numpy((words >> u32(8)).astype(np.float32) * np.float32(2.0 ** -24) >= np.float32(case["p"])).cuda()
    y = s["x"].double() * kept / (1 - float(np.float32(case["p"])))
    return dict(y=y if s["residual"] is None else y + s["residual"].double())
