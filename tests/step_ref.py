"""Plain 64-bit forms of the operators between ids and logits, for their tests."""
import numpy as np

import d3s_workloads as W
import train_ref as R

U, BF16 = R.U, R.BF16


def half_step(dtype):
    """an output's rounding, relative to its value"""
    return U if dtype == "f32" else BF16


# ---- verification ----
def probs(l, T):
    """softmax(l / T) along the last axis; zeros where all is masked"""
    T = np.maximum(np.float64(T), np.float64(np.float32(1e-5)))
    with np.errstate(all="ignore"):
        d = (l - l.max(-1, keepdims=True)) / T
        e = np.where(np.isneginf(l), 0.0, np.exp(d))
        S = e.sum(-1, keepdims=True)
        return np.where(S > 0, e / S, 0.0)


def draw(w, u):
    """the least j with w_0 + .. + w_j > u Z"""
    c = np.cumsum(w)
    at = np.nonzero(c > u * c[-1])[0]
    return int(at[0]) if len(at) else int(np.nonzero(w > 0)[0][-1])


def race(w, u):
    with np.errstate(all="ignore"):
        s = np.where(w > 0, np.maximum(w / -np.log(1 - u), -1.0), -2.0)
    return int(np.argmax(s))


def refused_row(l, T):
    return bool(np.isnan(l).any() or np.isposinf(l).any() or not np.isfinite(T))


def verify(target, draft, drafted, lengths, T, Td, u_accept, u_draw):
    """target [n, L + 1, V], draft [n, L, V] or None, T and Td [n]: (tokens, accepted,
    accept, sequences refused, sequences that drew from a masked row)"""
    n, L1, V = target.shape
    L = L1 - 1
    tokens, n_acc = np.full((n, L1), -1), np.zeros(n, int)
    accept = np.zeros((n, L))
    bad = masked = 0
    for b in range(n):
        m = L if lengths is None else min(max(int(lengths[b]), 0), L)
        rows = [(target[b, i], None if draft is None else draft[b, i]) for i in range(m)]
        ps, qs, ref = [], [], []
        for i, (t, d) in enumerate(rows):
            x = int(drafted[b, i])
            r = refused_row(t, T[b]) or (d is not None and refused_row(d, Td[b]))
            ref.append(r)
            inside = 0 <= x < V
            ps.append(0.0 if r or not inside else probs(t, T[b])[x])
            qs.append(1.0 if d is None else 0.0 if r or not inside else probs(d, Td[b])[x])
            accept[b, i] = np.nan if r else min(1.0, ps[i] / qs[i]) if qs[i] > 0 else float(ps[i] > 0)
        i, rejected, stop = 0, False, False
        while i < m:
            if ref[i]:
                stop = True
                break
            if not u_accept[b, i] * qs[i] < ps[i]:
                rejected = True
                break
            i += 1
        n_acc[b] = i
        tokens[b, :i] = drafted[b, :i]
        if stop or (i == m and refused_row(target[b, i], T[b])):
            bad += 1
            continue
        p = probs(target[b, i], T[b])
        if p.sum() == 0:
            masked += 1
            tokens[b, i] = 0
            continue
        w = p
        if rejected:
            q = np.zeros(V)
            if draft is not None:
                q = probs(draft[b, i], Td[b])
            elif 0 <= drafted[b, i] < V:
                q[drafted[b, i]] = 1.0
            w = np.maximum(p - q, 0)
            if w.sum() == 0:
                w = p
        tokens[b, i] = draw(w, float(u_draw[b]))
    return tokens, n_acc, accept, bad, masked


def keep_off_borders(target, draft, drafted, T, Td, u_accept):
    """u_accept with the draws moved that lie within 1e-4 of p / q, where rounding may
    decide (p and q are off by a few times 2^-24 of their exponents, below 30 here)"""
    n, L = drafted.shape
    out = u_accept.copy()
    V = target.shape[2]
    for b in range(n):
        for i in range(L):
            x = drafted[b, i]
            if not 0 <= x < V or refused_row(target[b, i], T[b]) or (draft is not None and refused_row(draft[b, i], Td[b])):
                continue
            p = probs(target[b, i], T[b])[x]
            q = 1.0 if draft is None else probs(draft[b, i], Td[b])[x]
            if q > 0 and abs(out[b, i] - p / q) < 1e-4:
                out[b, i] = out[b, i] + 2.0 ** -10 if out[b, i] < 0.5 else out[b, i] - 2.0 ** -10
    return out


# ---- embedding ----
def table_rows(n_ids, vocab, slot_rows):
    return vocab + (n_ids - 1) * slot_rows


def embed(ids, table, vocab, slot_rows, scale):
    """(y, the sum of its terms' sizes)"""
    n, t = ids.shape
    y, size = np.zeros((n, table.shape[1])), np.zeros((n, table.shape[1]))
    for k in range(t):
        live = (ids[:, k] >= 0) & (ids[:, k] < vocab)
        rows = table[ids[live, k] + k * slot_rows]
        y[live] += rows
        size[live] += np.abs(rows)
    return y * scale, size * abs(scale)


def embed_grad(ids, dy, vocab, slot_rows, scale):
    """(grad, the sum of its terms' sizes, their number a row)"""
    n, t = ids.shape
    rows = table_rows(t, vocab, slot_rows)
    g, size, count = np.zeros((rows, dy.shape[1])), np.zeros((rows, dy.shape[1])), np.zeros(rows)
    for k in range(t):
        live = (ids[:, k] >= 0) & (ids[:, k] < vocab)
        at = ids[live, k] + k * slot_rows
        np.add.at(g, at, dy[live])
        np.add.at(size, at, np.abs(dy[live]))
        np.add.at(count, at, 1)
    return g * scale, size * abs(scale), count


# ---- norm ----
def norm(h, gain, eps):
    with np.errstate(all="ignore"):
        rstd = 1 / np.sqrt((h * h).mean(1) + eps)
        return h * rstd[:, None] * gain, rstd


def norm_steps(width):
    """how many steps of 2^-24 rstd may be off, relative to itself: half of its sum's
    (additions of positive terms, each square's own), the mean, the root and the quotient"""
    return R.adds(width) / 2 + 6


def norm_grad(dy, h, gain, rstd, dsum):
    """(dx, a bound on its error in fp32, dgain, the sum of its terms' sizes)"""
    width = h.shape[1]
    xhat = h * rstd[:, None]
    a = dy * gain
    mean = (a * xhat).mean(1, keepdims=True)
    size = np.abs(a * xhat).mean(1, keepdims=True)
    dx = rstd[:, None] * (a - xhat * mean)
    err = U * rstd[:, None] * (4 * np.abs(a) + np.abs(xhat) * (6 * np.abs(mean) + (R.adds(width) + 6) * size))
    if dsum is not None:
        dx = dx + dsum
        err = err + U * (np.abs(dx) + np.abs(dsum))
    return dx, err + 1e-37, (dy * xhat).sum(0), np.abs(dy * xhat).sum(0)


def e4m3_values():
    """the 256 values, NaN at 0x7f and 0xff"""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b >= 128, -v, v)


# ---- dropout ----
def uniforms(n, seed, draw):
    """the first n of d3s_uniform_fill's, by numpy"""
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    words = W.philox4x32_10([(q & np.uint64(0xffffffff)).astype(np.uint32), (q >> np.uint64(32)).astype(np.uint32),
                             np.full(len(q), draw & 0xffffffff, np.uint32), np.full(len(q), draw >> 32, np.uint32)],
                            seed & 0xffffffff, seed >> 32)
    w = np.stack(words, 1).reshape(-1)[:n]
    return (w >> np.uint32(8)).astype(np.float32) * np.float32(2.0 ** -24)


def dropout(x, p, seed, draw, residual):
    """(y, the kept places)"""
    p = float(np.float32(p))
    kept = uniforms(x.size, seed, draw).reshape(x.shape).astype(np.float64) >= p
    y = np.where(kept, x / (1 - p) if p < 1 else 0.0, 0.0)
    return (y if residual is None else y + residual), kept
