"""The scoring and training operators as their callers issue them, for timing:
log probabilities of given tokens (with entropy and top alternatives) and their
gradient, dense layers with their epilogue and gradients, and the global
gradient norm with clipping.

A case is a dict of plain values:
  kind     "score" (d3s_logprob), "score_grad" (d3s_logprob_backward),
           "dense" (d3s_dense_bf16: y = residual + act(x w^T + bias)),
           "input_grad" (dx = dz w) and "weight_grad" (dw = old + dz^T x), both
           d3s_dense_bf16 with operands read transposed,
           "act_grad" (d3s_dense_activation_backward_bf16) or
           "clip" (d3s_clip_grads)
  rows, vocab, dtype, pad   the logits (pad: elements between two rows)
  tokens   given tokens a row; top: alternatives a row; per_row: a temperature
           for each row; banned: index 0 banned on half of the rows; entropy:
           the gradient has an entropy term
  m, n, k  a product's rows, outputs and inner length; act, bias, residual,
           keep (the pre-activation is kept), out ("bf16" / "f32")
  sizes    "heads" (weights of a model's heads), "ragged" (tensors from one
           element up) with count and total; clipped: the norm passes its limit

The widths 2048, 4096, 4097 and 151936 are those of d3s_workloads.py and
bench.py, the others generic.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

MIN_T = 1e-5
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _d3s():
    if "d3s" not in sys.modules:
        sys.path.insert(0, os.path.abspath("drama3-mlx_amd"))
    import d3s
    return d3s


def _score(name, rows, vocab, dtype, tokens, top, per_row, banned, kind="score", entropy=True, pad=0):
    return dict(name=name, kind=kind, rows=rows, vocab=vocab, dtype=dtype, pad=pad, tokens=tokens, top=top,
                per_row=per_row, banned=banned, entropy=entropy)


def _dense(name, m, n, k, act="none", bias=False, residual=False, keep=False, out="bf16", kind="dense", pad=0):
    return dict(name=name, kind=kind, m=m, n=n, k=k, act=act, bias=bias, residual=residual, keep=keep, out=out,
                pad=pad)


def listed():
    return [
        # the main token of one stream, scored after its draw, with five alternatives
        _score("score_token", 1, 4097, "bf16", 1, 5, False, False),
        # a serving step over a text vocabulary: the drawn token and twenty alternatives
        _score("score_text", 64, 151936, "bf16", 1, 20, True, False),
        # the tokens of a rollout scored for training: inputs far past every cache
        _score("score_rollout", 4096, 151936, "bf16", 1, 0, False, False),
        # the codebook heads' loss: fp32 logits, per-row temperatures, eos banned on some rows
        _score("grad_codebooks", 4096, 4097, "f32", 1, 0, True, True, kind="score_grad"),
        # a rollout's loss over a text vocabulary
        _score("grad_rollout", 2048, 151936, "bf16", 1, 0, False, False, kind="score_grad"),
        # an adapter before the heads, one stream's next frame
        _dense("dense_frame", 1, 2048, 2048, "silu", True, True),
        # the same adapter over a batch of prompts, its pre-activation kept for the backward
        _dense("dense_prompt", 8192, 2048, 2048, "gelu", True, True, True),
        # the backbone head's input gradient: rows of 4097 padded to whole 16 bytes
        _dense("input_grad", 8192, 2048, 4097, kind="input_grad", pad=7),
        # its weight gradient, added to an earlier micro-batch's: rows of 4097 one after the other
        _dense("weight_grad", 4097, 2048, 8192, residual=True, out="f32", kind="weight_grad"),
        # the adapter's activation and bias gradient
        _dense("act_grad", 8192, 2048, 0, "silu", True, kind="act_grad"),
        # the ten heads' weight gradients, clipped
        dict(name="clip_heads", kind="clip", sizes="heads", count=10, total=10 * 4097 * 2048, dtype="f32", clipped=True),
        # a small model's many tensors, most of them short
        dict(name="clip_ragged", kind="clip", sizes="ragged", count=150, total=2000000, dtype="mixed", clipped=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "score", "score_grad", "dense", "dense", "input_grad", "weight_grad", "act_grad", "clip"])
    if kind in ("score", "score_grad"):
        vocab = rng.choice([4096, 4097, 151936, _log(rng, 1, 200000), _log(rng, 1, 200000)])
        rows = _log(rng, 1, min(8192, max(1, 300000000 // vocab)))
        top = rng.choice([0, 0, 1, 5, 20, rng.randint(1, 64)]) if kind == "score" and rows * vocab < 60000000 else 0
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(["bf16", "f32"]),
                    pad=rng.choice([0, 0, rng.randint(1, 9)]), tokens=rng.choice([1, 1, 1, rng.randint(2, 16)]),
                    top=min(top, vocab), per_row=rng.random() < 0.5, banned=vocab > 1 and rng.random() < 0.3,
                    entropy=rng.random() < 0.7)
    if kind == "clip":
        sizes = rng.choice(["heads", "ragged", "ragged"])
        count = rng.randint(1, 12) if sizes == "heads" else _log(rng, 1, 900)
        total = count * 4097 * 2048 if sizes == "heads" else _log(rng, max(count, 1000), 60000000)
        return dict(kind=kind, sizes=sizes, count=count, total=total, dtype=rng.choice(["f32", "bf16", "mixed"]),
                    clipped=rng.random() < 0.7)
    size = lambda: rng.choice([2048, 4096, 4097, _log(rng, 16, 8192), 8 * _log(rng, 2, 1024)])  # noqa: E731
    most = 8192 * 2048 * 4097  # multiply-adds of the largest listed product
    if kind == "dense":
        n, k = size(), size()
        m = _log(rng, 1, rng.choice([64, min(8192, most // (n * k))]))
        return dict(kind=kind, m=m, n=n, k=k, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.6, residual=rng.random() < 0.5, keep=rng.random() < 0.3,
                    out=rng.choice(["bf16", "bf16", "f32"]), pad=rng.choice([0, 0, 8, rng.randint(1, 15)]))
    rows = _log(rng, 16, 8192)
    if kind == "act_grad":
        return dict(kind=kind, m=rows, n=size(), k=0, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.7, residual=False, keep=False, out="bf16", pad=rng.choice([0, 0, rng.randint(1, 15)]))
    pad = rng.choice([0, 0, 7, rng.randint(1, 15)])
    if kind == "input_grad":
        n, k = size(), size()
        return dict(kind=kind, m=min(rows, most // (n * k)), n=n, k=k, act="none", bias=False,
                    residual=rng.random() < 0.3, keep=False, out=rng.choice(["bf16", "f32"]), pad=pad)
    m, n = size(), size()
    return dict(kind=kind, m=m, n=n, k=min(rows, most // (m * n)), act="none", bias=False, residual=rng.random() < 0.6,
                keep=False, out=rng.choice(["f32", "f32", "bf16"]), pad=pad)


def _rows(shape, pad, dtype, g, scale=1.0):
    """a matrix whose rows lie `pad` elements apart"""
    t = torch.empty(shape[0], shape[1] + pad, dtype=dtype, device="cuda").normal_(0, scale, generator=g)
    return t[:, :shape[1]]


def _clip_sizes(case):
    if case["sizes"] == "heads":
        return [case["total"] // case["count"]] * case["count"]
    rng = np.random.default_rng([case["total"], case["count"]])
    w = np.exp(rng.normal(0, 2.0, case["count"]))  # a few long tensors, many short ones
    return [max(1, int(v)) for v in w / w.sum() * case["total"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        rows, vocab, dt = case["rows"], case["vocab"], DT[case["dtype"]]
        logits = _rows((rows, vocab), case["pad"], dt, g, 2.5)
        at = torch.randint(0, vocab, (rows, min(8, vocab)), device="cuda", generator=g)
        up = torch.rand(at.shape, device="cuda", generator=g) * 6 + 4
        logits.scatter_(1, at, up.to(dt))  # a few likely tokens
        s["logits"] = logits
        pick = torch.randint(0, at.shape[1], (rows, case["tokens"]), device="cuda", generator=g)
        tokens = at.gather(1, pick)  # drawn tokens are mostly likely ones
        r = torch.rand(tokens.shape, device="cuda", generator=g)
        tokens = torch.where(r < 0.3, torch.randint(0, vocab, tokens.shape, device="cuda", generator=g), tokens)
        s["tokens"] = torch.where(r > 0.95, -1, tokens).to(torch.int32)  # padding
        s["T"] = torch.rand(rows, device="cuda", generator=g) * 0.7 + 0.5 if case["per_row"] else None
        s["banned"] = None
        if case["banned"]:
            s["banned"] = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.5, 0, -1).to(torch.int32)
        new = lambda shape, t: torch.empty(shape, dtype=t, device="cuda")  # noqa: E731
        if kind == "score":
            s["out"] = dict(logprobs=new((rows, case["tokens"]), torch.float32), stats=new((rows, 2), torch.float32))
            if case["entropy"]:
                s["out"]["entropy"] = new((rows,), torch.float32)
            if case["top"]:
                s["out"]["top_ids"] = new((rows, case["top"]), torch.int32)
                s["out"]["top_logprobs"] = new((rows, case["top"]), torch.float32)
        else:
            # what the forward pass left: each row's greatest logit, its sum and its entropy
            s["stats"], s["entropy"] = _row_sums(s, torch.float64)
            s["grad_logprobs"] = torch.randn(rows, case["tokens"], device="cuda", generator=g)
            s["grad_entropy"] = torch.full((rows,), 0.01, device="cuda") if case["entropy"] else None
            s["out"] = dict(grad=new((rows, vocab), dt))
    elif kind == "clip":
        sizes = _clip_sizes(case)
        bf16 = [case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 3 == 0) for i in range(len(sizes))]
        # gradients lie in one block a type, as a bucketed backward leaves them
        s["grads"], s["out"] = {}, {}
        src, dst = [0] * len(sizes), [0] * len(sizes)
        for name, dt, mine in (("f32", torch.float32, False), ("bf16", torch.bfloat16, True)):
            total = sum(n for n, b in zip(sizes, bf16) if b == mine)
            if total:
                s["grads"][name] = _rows((1, total), 0, dt, g, 0.02)[0]
                s["out"][name] = torch.empty(total, dtype=dt, device="cuda")
                at = 0
                for i, n in enumerate(sizes):
                    if bf16[i] == mine:
                        src[i] = s["grads"][name][at:].data_ptr()
                        dst[i] = s["out"][name][at:].data_ptr()
                        at += n
        s["src"], s["dst"] = np.array(src, np.uint64), np.array(dst, np.uint64)
        s["numel"] = np.array(sizes, np.int64)
        s["dtypes"] = np.array([1 if b else 0 for b in bf16], np.int32)
        s["max_norm"] = 1.0 if case["clipped"] else 1e6
        s["norm"] = torch.empty((), dtype=torch.float32, device="cuda")
    else:
        m, n, k, pad = case["m"], case["n"], case["k"], case["pad"]
        out = DT[case["out"]]
        bf = torch.bfloat16
        s["bias"] = torch.empty(n, dtype=bf, device="cuda").normal_(0, 0.5, generator=g) if case["bias"] else None
        s["residual"] = _rows((m, n), 0, out, g) if case["residual"] else None
        s["out"] = dict(y=torch.empty(m, n, dtype=out, device="cuda"))
        if case["keep"]:
            s["out"]["z"] = torch.empty(m, n, dtype=bf, device="cuda")
        if kind == "dense":
            s["x"], s["w"] = _rows((m, k), pad, bf, g), _rows((n, k), pad, bf, g, k ** -0.5)
        elif kind == "input_grad":  # y [m, n] = dz [m, k] w [k, n]
            s["x"], s["w"] = _rows((m, k), pad, bf, g), _rows((k, n), 0, bf, g, k ** -0.5)
        elif kind == "weight_grad":  # y [m, n] = dz^T x with dz [k, m], x [k, n]
            s["x"], s["w"] = _rows((k, m), pad, bf, g), _rows((k, n), 0, bf, g, k ** -0.5)
        else:
            s["dy"], s["z"] = _rows((m, n), pad, bf, g), _rows((m, n), 0, bf, g)
            s["out"] = dict(dz=torch.empty(m, n, dtype=bf, device="cuda"))
            if case["bias"]:
                s["out"]["dbias"] = torch.empty(n, dtype=torch.float32, device="cuda")
    return s


# ---- the plain forms: elementary operations in 32 bits ----
def _scaled(s, dt):
    """(logits with the banned index out, masked places, temperatures) in dt"""
    x = s["logits"].to(dt, copy=s["banned"] is not None)
    if s["banned"] is not None:
        x[:, 0] = torch.where(s["banned"] == 0, -math.inf, x[:, 0])
    T = s["T"].to(dt)[:, None].clamp_min(MIN_T) if s["T"] is not None else torch.ones((), dtype=dt, device="cuda")
    return x, x == -math.inf, T


def _row_sums(s, dt):
    """([rows, 2]: the greatest logit and log sum exp((l - greatest) / T); the entropy), fp32"""
    step = max(1, (256 << 20) // s["case"]["vocab"])
    stats, entropy = [], []
    for r in range(0, s["case"]["rows"], step):
        part = dict(logits=s["logits"][r:r + step], banned=None if s["banned"] is None else s["banned"][r:r + step],
                    T=None if s["T"] is None else s["T"][r:r + step])
        x, masked, T = _scaled(part, dt)
        top = x.amax(1, keepdim=True)
        d = x.sub_(top).div_(T).masked_fill_(masked, 0)
        e = d.exp().masked_fill_(masked, 0)
        S = e.sum(1)
        entropy.append((S.log() - e.mul_(d).sum(1) / S).float())
        stats.append(torch.stack([top[:, 0], S.log()], 1).float())
    return torch.cat(stats), torch.cat(entropy)


def _plain_score(s):
    case, out = s["case"], {}
    x, masked, T = _scaled(s, torch.float32)
    top = x.amax(1, keepdim=True)
    d = (x - top) / T
    zero = d.masked_fill(masked, 0)
    e = zero.exp().masked_fill_(masked, 0)
    S = e.sum(1, keepdim=True)
    logp = lambda ids: d.gather(1, ids) - S.log()  # noqa: E731
    tokens = s["tokens"].long()
    out["logprobs"] = torch.where(tokens < 0, 0.0, logp(tokens.clamp_min(0)))
    out["stats"] = torch.cat([top, S.log()], 1)
    if case["entropy"]:
        out["entropy"] = S.log()[:, 0] - (e * zero).sum(1) / S[:, 0]
    if case["top"]:
        ids = x.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), logp(ids)
    return out


def _plain_score_grad(s):
    x, masked, T = _scaled(s, torch.float32)
    logp = (x - s["stats"][:, :1]) / T - s["stats"][:, 1:]
    p = logp.exp()
    tokens, g = s["tokens"].long(), s["grad_logprobs"]
    g = torch.where(tokens < 0, 0.0, g)
    dx = -p * g.sum(1, keepdim=True)
    if s["grad_entropy"] is not None:
        dx -= s["grad_entropy"][:, None] * p * (logp.masked_fill(masked, 0) + s["entropy"][:, None])
    dx.scatter_add_(1, tokens.clamp_min(0), g)
    return dict(grad=(dx / T).masked_fill_(masked, 0).to(s["logits"].dtype))


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + (-z).exp())
    if act == "gelu":
        return z * 0.5 * (1 + (z * 0.5 ** 0.5).erf())
    if act == "gelu_tanh":
        return z * 0.5 * (1 + ((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)).tanh())
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        f = 1 / (1 + (-z).exp())
        return f * (1 + z * (1 - f))
    if act == "gelu":
        return 0.5 * (1 + (z * 0.5 ** 0.5).erf()) + z * (-0.5 * z * z).exp() * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = (c * (z + 0.044715 * z ** 3)).tanh()
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_dense(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    z = x.t() @ w if case["kind"] == "weight_grad" else x @ w if case["kind"] == "input_grad" else x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(y=y.to(DT[case["out"]]))
    if case["keep"]:
        out["z"] = z.to(torch.bfloat16)
    return out


def _plain_act_grad(s):
    dz = s["dy"].float() * _act_slope(s["z"].float(), s["case"]["act"])
    out = dict(dz=dz.to(torch.bfloat16))
    if s["case"]["bias"]:
        out["dbias"] = dz.sum(0)
    return out


def _plain_clip(s):
    grads = {name: g.float() for name, g in s["grads"].items()}
    norm = sum(g.double().square().sum() for g in grads.values()).sqrt().float()
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
    out = {name: (g * scale).to(s["grads"][name].dtype) for name, g in grads.items()}
    out["norm"] = norm
    return out


# ---- the framework's calls ----
def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    d3s, case, out = _d3s(), s["case"], s["out"]
    stream = torch.cuda.current_stream().cuda_stream or None
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        logits = s["logits"]
        T = 1.0 if s["T"] is None else ("ptr", s["T"].data_ptr())
        common = (logits.data_ptr(), d3s.DTYPE_F32 if case["dtype"] == "f32" else d3s.DTYPE_BF16, case["rows"],
                  case["vocab"], case["vocab"] + case["pad"], T, _ptr(s["banned"]), s["tokens"].data_ptr(), case["tokens"])
        if kind == "score":
            rc = d3s.logprob_raw(*common, out["logprobs"].data_ptr(), _ptr(out.get("entropy")), out["stats"].data_ptr(),
                                 case["top"], _ptr(out.get("top_ids")), _ptr(out.get("top_logprobs")), stream=stream)
        else:
            rc = d3s.logprob_backward_raw(*common, s["stats"].data_ptr(), s["entropy"].data_ptr(),
                                          s["grad_logprobs"].data_ptr(), _ptr(s["grad_entropy"]),
                                          out["grad"].data_ptr(), case["vocab"], stream=stream)
    elif kind == "clip":
        rc = d3s.clip_grads_raw(s["src"].ctypes.data, s["dst"].ctypes.data, s["numel"].ctypes.data,
                                s["dtypes"].ctypes.data, len(s["numel"]), s["max_norm"], s["norm"].data_ptr(),
                                stream=stream)
        out = dict(out, norm=s["norm"])
    elif kind == "act_grad":
        n = case["n"]
        rc = d3s.dense_activation_backward_raw(s["dy"].data_ptr(), n + case["pad"], s["z"].data_ptr(), n, case["m"], n,
                                               d3s.ACTIVATIONS[case["act"]], out["dz"].data_ptr(), n,
                                               _ptr(out.get("dbias")), stream=stream)
    else:
        x, w = s["x"], s["w"]
        rc = d3s.dense_raw(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), case["m"], case["n"], case["k"],
                           out["y"].data_ptr(), case["n"],
                           d3s.DTYPE_F32 if case["out"] == "f32" else d3s.DTYPE_BF16,
                           x_transposed=kind == "weight_grad", w_transposed=kind != "dense", bias=_ptr(s["bias"]),
                           activation=d3s.ACTIVATIONS[case["act"]], residual=_ptr(s["residual"]),
                           residual_stride=case["n"], z=_ptr(out.get("z")), z_stride=case["n"], stream=stream)
    if rc != d3s.OK:
        raise RuntimeError(f"{kind}: status {rc}")
    return out


def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    return {"score": _plain_score, "score_grad": _plain_score_grad, "clip": _plain_clip,
            "act_grad": _plain_act_grad}.get(kind, _plain_dense)(s)


def work(case):
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        rows, vocab, size = case["rows"], case["vocab"], 4 if case["dtype"] == "f32" else 2
        a_row = 8 * case["tokens"] + 8 * case["top"] + 12 + 4 * case["per_row"] + 4 * case["banned"]
        return {"bytes": rows * (vocab * size * (2 if kind == "score_grad" else 1) + a_row), "flops": 8 * rows * vocab}
    if kind == "clip":
        size = {"f32": 4, "bf16": 2, "mixed": 3.33}[case["dtype"]]
        return {"bytes": 2 * case["total"] * size, "flops": 3 * case["total"]}
    m, n, k, size = case["m"], case["n"], case["k"], 4 if case["out"] == "f32" else 2
    if kind == "act_grad":
        return {"bytes": 6 * m * n + 4 * n * case["bias"], "flops": 12 * m * n}
    return {"bytes": 2 * (m * k + n * k) + m * n * (size * (1 + case["residual"]) + 2 * case["keep"]) + 2 * n * case["bias"],
            "flops": 2 * m * n * k}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("score", "score_grad"):
        return _exact_rows(s)
    if kind == "clip":
        norm = sum(float(g.double().pow(2).sum()) for g in s["grads"].values()) ** 0.5
        c = min(1.0, s["max_norm"] / norm)
        return {**{name: g.double() * c for name, g in s["grads"].items()}, "norm": norm}
    f = {"none": lambda v: v, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
    if kind == "act_grad":
        z = s["z"].double().requires_grad_()
        dz, = torch.autograd.grad(f(z), z, s["dy"].double())
        return {"dz": dz, "dbias": dz.sum(0)} if case["bias"] else {"dz": dz}
    if 2 * case["m"] * case["n"] * case["k"] > 6e11:
        return None
    x, w = s["x"].double(), s["w"].double()
    x = x.t() if kind == "weight_grad" else x
    z = torch.mm(x, w.t() if kind == "dense" else w)
    z = z if s["bias"] is None else z.add(s["bias"])
    y = f(z) if s["residual"] is None else f(z).add(s["residual"])
    return {"y": y, "z": z} if case["keep"] else {"y": y}


def _exact_rows(s):
    """log-softmax by torch in 64 bits, the gradient from its Jacobian, a block of rows at a time"""
    case, parts = s["case"], []
    for r in range(0, case["rows"], max(1, (100 << 20) // case["vocab"])):
        at = slice(r, r + max(1, (100 << 20) // case["vocab"]))
        l = s["logits"][at].double()  # noqa: E741
        if s["banned"] is not None:
            l[s["banned"][at] == 0, 0] = -math.inf
        T = s["T"][at].double()[:, None].clamp_min(MIN_T) if s["T"] is not None else 1.0
        logp = torch.log_softmax(l / T, 1)
        dead = torch.isneginf(logp)
        p, tok = logp.exp(), s["tokens"][at].long()
        live = tok >= 0
        H = -(p * logp.masked_fill(dead, 0)).sum(1)
        if case["kind"] == "score_grad":
            g = s["grad_logprobs"][at].double() * live
            dx = torch.zeros_like(p).scatter_add_(1, tok.clamp_min(0), g) - g.sum(1, keepdim=True) * p
            if case["entropy"]:
                dx -= s["grad_entropy"][at].double()[:, None] * p * (logp.masked_fill(dead, 0) + H[:, None])
            parts.append({"grad": dx.div(T).masked_fill(dead, 0)})
            continue
        most = l.amax(1)
        part = {"logprobs": logp.gather(1, tok.clamp_min(0)) * live,
                "stats": torch.stack([most, torch.logsumexp((l - most[:, None]) / T, 1)], 1)}
        if case["entropy"]:
            part["entropy"] = H
        if case["top"]:
            part["top_logprobs"] = logp.gather(1, torch.argsort(l, dim=1, descending=True, stable=True)[:, :case["top"]])
        parts.append(part)
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    return {**out, "top_ids": None} if case["top"] else out
