"""Plain 64-bit forms of the scoring and training operators, and device helpers
for their tests.  u is half a step of fp32; a bf16 result may be half a step,
2^-8 of its value, off."""
import math

import numpy as np

import d3s_workloads as W

U = 2.0 ** -24
BF16 = 2.0 ** -8


def to_bits(x, dtype):
    """x as the library's array of dtype "f32" / "bf16"; and its values in float64"""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return np.ascontiguousarray(x), x.astype(np.float64)
    bits = np.empty(x.shape, np.uint16)
    nan = np.isnan(x)
    with np.errstate(invalid="ignore"):
        bits[...] = W.f32_to_bf16_bits(np.where(nan, 0, x))
    bits[nan] = 0x7fc0
    return bits, from_bits(bits)


def from_bits(b):
    return W.bf16_bits_to_f32(b).astype(np.float64) if b.dtype == np.uint16 else b.astype(np.float64)


def with_stride(bits, stride, offset=0, fill=0):
    """(flat array of the rows `stride` apart after `offset` elements; the rest `fill`)"""
    n, v = bits.shape
    flat = np.full(offset + (n - 1) * stride + v if n else offset, fill, bits.dtype)
    for r in range(n):
        flat[offset + r * stride: offset + r * stride + v] = bits[r]
    return flat


def rows_at(flat, n, v, stride, offset=0):
    return np.stack([flat[offset + r * stride: offset + r * stride + v] for r in range(n)]) if n else \
        np.empty((0, v), flat.dtype)


def score(l, T, banned, tokens, n_top):
    """l float64 [n, V], T float64 [n], banned int [n] or None, tokens int [n, t]"""
    l = l.copy()
    n, V = l.shape
    if banned is not None:
        for r in range(n):
            if 0 <= banned[r] < V:
                l[r, banned[r]] = -math.inf
    T = np.maximum(T, np.float64(np.float32(1e-5)))[:, None]
    with np.errstate(all="ignore"):
        m = l.max(1, keepdims=True)
        d = np.where(np.isneginf(l), -math.inf, (l - m) / T)
        e = np.exp(d)
        S = e.sum(1, keepdims=True)
        logS = np.log(S)
        logp = d - logS
        live = e > 0
        ed = np.where(live, e * np.where(live, d, 0), 0).sum(1) / S[:, 0]
        H = logS[:, 0] - ed
    refused = np.isnan(l).any(1) | np.isposinf(l).any(1) | ~np.isfinite(T[:, 0])
    masked = ~refused & np.isneginf(l).all(1)
    logp[masked], H[masked], logS[masked], m[masked] = -math.inf, 0.0, -math.inf, -math.inf
    ed = np.where(masked, 0.0, ed)
    logp[refused], H[refused], logS[refused], m[refused] = (math.nan,) * 4
    logp[logp < -np.finfo(np.float32).max] = -math.inf  # outside fp32: the result is its infinity
    none = (tokens < 0) | (tokens >= V)
    lp = np.take_along_axis(logp, np.where(none, 0, tokens), 1)
    lp = np.where(none & ~refused[:, None], 0.0, lp)
    order = np.argsort(-l, axis=1, kind="stable")[:, :n_top]
    order[masked] = np.arange(n_top)
    top_lp = np.take_along_axis(logp, order, 1)
    order[refused] = -1
    return dict(l=l, T=T, d=d, logp=logp, m=m[:, 0], logS=logS[:, 0], H=H, Ed=-ed, logprobs=lp, top_ids=order,
                top_logprobs=top_lp, refused=refused, masked=masked, none=none)


def adds(V):
    """additions in a row's longest chain: a lane's terms, the trees, the exponential's own steps"""
    return V / 256 + 64


def score_tol(ref, logp):
    """of a log probability: the difference and its quotient, the logarithm of the
    sum (its terms' exponents are rounded relative to themselves)"""
    V = ref["l"].shape[1]
    logS = np.abs(np.where(np.isfinite(ref["logS"]), ref["logS"], 0))[:, None]
    Ed = np.where(np.isfinite(ref["Ed"]), ref["Ed"], 0)[:, None]
    lp = np.where(np.isfinite(logp), np.abs(logp), 0)
    return U * (4 * (lp + logS) + 4 * Ed + adds(V))


def entropy_tol(ref):
    V = ref["l"].shape[1]
    Ed = np.where(np.isfinite(ref["Ed"]), ref["Ed"], 0)
    logS = np.abs(np.where(np.isfinite(ref["logS"]), ref["logS"], 0))
    return U * (adds(V) * (1 + 2 * Ed) + 4 * logS + 4 * Ed * Ed)


def score_grad(ref, tokens, g, gH):
    """(the gradient, a bound on its error in fp32)"""
    n, V = ref["l"].shape
    g = np.where(ref["none"], 0.0, g)
    G = g.sum(1, keepdims=True)
    gH = np.zeros((n, 1)) if gH is None else gH[:, None].astype(np.float64)
    with np.errstate(all="ignore"):
        p = np.exp(ref["logp"])
        lp = np.where(p > 0, ref["logp"], 0)
        H, logS = ref["H"][:, None], ref["logS"][:, None]
        dx = -p * (G + gH * (lp + H))
        size = p * (np.abs(g).sum(1, keepdims=True) + np.abs(gH) * (np.abs(lp) + H + 1 + np.abs(logS)))
        err = U * size * (64 + 8 * np.abs(lp) + 8 * np.abs(logS))
        for r in range(n):
            for t in range(tokens.shape[1]):
                if not ref["none"][r, t]:
                    dx[r, tokens[r, t]] += g[r, t]
                    err[r, tokens[r, t]] += U * tokens.shape[1] * 4 * np.abs(g[r]).sum()
        dx, err = dx / ref["T"], err / ref["T"]
    dead = np.isneginf(ref["l"])
    dx[dead], err[dead] = 0.0, 0.0
    return dx, err + 1e-37


def act(z, name):
    from scipy.special import erf
    with np.errstate(over="ignore"):
        if name == "relu":
            return np.maximum(z, 0)
        if name == "silu":
            return z / (1 + np.exp(-z))
        if name == "gelu":
            return 0.5 * z * (1 + erf(z / math.sqrt(2)))
        if name == "gelu_tanh":
            return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(z, name):
    from scipy.special import erf
    with np.errstate(over="ignore"):
        if name == "relu":
            return (z > 0).astype(np.float64)
        if name == "silu":
            f = 1 / (1 + np.exp(-z))
            return f * (1 + z * (1 - f))
        if name == "gelu":
            return 0.5 * (1 + erf(z / math.sqrt(2))) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        if name == "gelu_tanh":
            c = math.sqrt(2 / math.pi)
            t = np.tanh(c * (z + 0.044715 * z ** 3))
            return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return np.ones_like(z)


def assert_near(got, ref, tol, what=""):
    """got within tol of ref; infinities and NaN alike"""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    tol = np.broadcast_to(tol, ref.shape)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    odd = ~np.isfinite(ref)
    assert np.array_equal(got[odd & ~np.isnan(ref)], ref[odd & ~np.isnan(ref)]), what
    bad = ~(np.abs(got - ref) <= tol) & ~odd
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], ref[bad][:4], tol[bad][:4])


class Arena:
    """device arrays of one test, freed together"""

    def __init__(self):
        self.held = []

    def put(self, arr):
        import hiprt
        b = hiprt.to_device(arr)
        self.held.append(b)
        return b

    def room(self, nbytes, byte=None):
        import hiprt
        b = hiprt.DeviceBuffer(max(int(nbytes), 16))
        if byte is not None:
            hiprt.check(hiprt.hip().hipMemset(b.ptr, byte, b.nbytes))
        self.held.append(b)
        return b

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for b in self.held:
            b.free()
