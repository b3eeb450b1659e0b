"""ctypes binding of libd3sampler.so, the MI355X token sampler.

The host-side counterpart of the reference's ctypes layer for this path
(tests/d3.py:211-217 binds d3_sample of src/testapi.c:155-166).  It loads the
in-tree library and fails loudly when it is missing: there is no CPU fallback.
"""
import ctypes
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libd3sampler.so")

DTYPE_F32 = 0
DTYPE_BF16 = 1
DTYPE_E4M3 = 2  # outputs of rms_norm_raw only
FLAG_GENERIC = 1
FLAG_EXACT_LSE = 2
FLAG_EXACT_SELECT = 4
FLAG_OP_GRAPH = 8
FLAG_ONE_LAUNCH = 16
COUNTER_REFUSED, COUNTER_ALL_MASKED, COUNTER_EXACT_SELECT, COUNTER_EXACT_LSE = range(4)
NUM_COUNTERS = 4
OK = 0
ERR_ARG = -1
ERR_UNSUPPORTED = -2
ERR_SCRATCH = -6
ERR_WORKSPACE = -7
SCRATCH_BYTES = 4 << 20
MAX_VOCAB = (1 << 24) - 1
MAX_TOKENS = 64
MAX_TOP = 64
MAX_DRAFT = 64
MAX_RANKED = 1024
MAX_IDS = 64
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}  # D3S_ACT_*

_lib = None


class RasParams(ctypes.Structure):
    """d3s_ras_params (include/d3s_sampler.h)"""
    _fields_ = [("temperature", ctypes.c_float), ("top_p", ctypes.c_float), ("top_k", ctypes.c_int),
                ("retry_temperature", ctypes.c_float), ("retry_top_p", ctypes.c_float),
                ("retry_top_k", ctypes.c_int), ("eos_id", ctypes.c_int32),
                ("semantic_start", ctypes.c_int32), ("semantic_end", ctypes.c_int32),
                ("code_vocab", ctypes.c_int32)]


class DenseParams(ctypes.Structure):
    """d3s_dense_params (include/d3s_train.h)"""
    _fields_ = [("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("x_transposed", ctypes.c_int),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("w_transposed", ctypes.c_int),
                ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64), ("bias", ctypes.c_void_p),
                ("activation", ctypes.c_int), ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64),
                ("z", ctypes.c_void_p), ("z_stride", ctypes.c_int64), ("y", ctypes.c_void_p),
                ("y_stride", ctypes.c_int64), ("y_dtype", ctypes.c_int)]


class VerifyParams(ctypes.Structure):
    """d3s_verify_params (include/d3s_step.h)"""
    _fields_ = [("target", ctypes.c_void_p), ("target_dtype", ctypes.c_int), ("target_stride", ctypes.c_int64),
                ("draft", ctypes.c_void_p), ("draft_dtype", ctypes.c_int), ("draft_stride", ctypes.c_int64),
                ("n_seqs", ctypes.c_int64), ("n_draft", ctypes.c_int), ("vocab", ctypes.c_int64),
                ("drafted", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("temperature", ctypes.c_void_p),
                ("temperature_scalar", ctypes.c_float), ("draft_temperature", ctypes.c_void_p),
                ("draft_temperature_scalar", ctypes.c_float), ("u_accept", ctypes.c_void_p), ("u_draw", ctypes.c_void_p),
                ("tokens", ctypes.c_void_p), ("n_accepted", ctypes.c_void_p), ("accept", ctypes.c_void_p),
                ("counters", ctypes.c_void_p)]


def ras_params(**kw):
    """RasParams from keyword fields; the retry defaults to the reference's
    RAS_TEMPERATURE / RAS_TOP_P / RAS_TOP_K (src/tower.c:13-16)."""
    d = dict(retry_temperature=1.0, retry_top_p=0.95, retry_top_k=30)
    d.update(kw)
    return RasParams(**d)


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C drama3-mlx_amd` "
                               "(or __graft_entry__.build()); there is no fallback")
        L = ctypes.CDLL(LIB_PATH)
        vp, i64, i32, f32, u32 = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float,
                                  ctypes.c_uint)
        L.d3s_sample.argtypes = [vp, i32, i64, i64, i64, vp, i32, vp, vp, f32, f32, vp, vp, vp, vp,
                                 vp, u32, vp]
        L.d3s_sample.restype = i32
        L.d3s_sample_noalloc.argtypes = [vp, i32, i64, i64, i64, vp, i32, vp, vp, f32, f32, vp, vp, vp, vp,
                                         vp, u32, vp]
        L.d3s_sample_noalloc.restype = i32
        L.d3s_sample_ws.argtypes = [vp, i32, i64, i64, i64, vp, i32, vp, vp, f32, f32, vp, vp, vp, vp,
                                    vp, u32, vp, i64, vp]
        L.d3s_sample_ws.restype = i32
        L.d3s_sample_seeded.argtypes = [vp, i32, i64, i64, i64, ctypes.c_uint64, ctypes.c_uint64, i32, vp, vp,
                                        f32, f32, vp, vp, vp, vp, vp, u32, vp]
        L.d3s_sample_seeded.restype = i32
        L.d3s_sample_workspace_bytes.argtypes = [i32, i64, i64, i32, u32]
        L.d3s_sample_workspace_bytes.restype = i64
        L.d3s_workspace_init.argtypes = [vp, i64, vp]
        L.d3s_workspace_init.restype = i32
        L.d3s_stream_workspace_release.argtypes = [vp]
        L.d3s_stream_workspace_release.restype = i32
        L.d3s_sample_ras_ws.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, i32,
                                        ctypes.POINTER(RasParams), vp, vp, vp, vp, vp, vp, i64, vp]
        L.d3s_sample_ras_ws.restype = i32
        L.d3s_sample_ras_workspace_bytes.argtypes = [i32, i64, i64, ctypes.POINTER(RasParams), i32]
        L.d3s_sample_ras_workspace_bytes.restype = i64
        L.d3s_linear_sample_bf16_ws.argtypes = [vp, vp, i64, i64, i64, vp, vp, i32, vp, vp, f32, f32, vp, vp,
                                                vp, vp, u32, vp, i64, vp]
        L.d3s_linear_sample_bf16_ws.restype = i32
        L.d3s_linear_sample_workspace_bytes.argtypes = [i64, i64, i64, i32, u32, i32]
        L.d3s_linear_sample_workspace_bytes.restype = i64
        L.d3s_sample_ras.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp, i32,
                                     ctypes.POINTER(RasParams), vp, vp, vp, vp, vp, vp]
        L.d3s_sample_ras.restype = i32
        L.d3s_linear_bf16.argtypes = [vp, vp, i64, i64, i64, vp, vp]
        L.d3s_linear_bf16.restype = i32
        L.d3s_linear_sample_bf16.argtypes = [vp, vp, i64, i64, i64, vp, vp, i32, vp, vp, f32, f32, vp, vp,
                                             vp, vp, u32, vp]
        L.d3s_linear_sample_bf16.restype = i32
        L.d3s_uniform_fill.argtypes = [vp, i64, ctypes.c_uint64, ctypes.c_uint64, vp]
        L.d3s_uniform_fill.restype = i32
        L.d3s_max_k.argtypes = []
        L.d3s_max_k.restype = i32
        L.d3s_fused_max_vocab.argtypes = [i32]
        L.d3s_fused_max_vocab.restype = i32
        L.d3s_math_selftest.argtypes = [vp, vp, vp, vp, vp, i64, f32, vp]
        L.d3s_math_selftest.restype = i32
        L.d3s_exp2_selftest.argtypes = [vp, vp, i64, vp]
        L.d3s_exp2_selftest.restype = i32
        L.d3s_log2_selftest.argtypes = [vp, vp, i64, vp]
        L.d3s_log2_selftest.restype = i32
        rows = [vp, i32, i64, i64, i64, vp, f32, vp, vp, i32]
        scores = rows + [vp, vp, vp, i32, vp, vp, vp]
        L.d3s_logprob.argtypes = scores + [vp]
        L.d3s_logprob_ws.argtypes = scores + [vp, i64, vp]
        L.d3s_logprob_workspace_bytes.argtypes = [i32, i64, i64, i32]
        L.d3s_logprob_backward.argtypes = rows + [vp, vp, vp, vp, vp, i64, vp]
        dense = ctypes.POINTER(DenseParams)
        L.d3s_dense_bf16.argtypes = [dense, vp]
        L.d3s_dense_bf16_ws.argtypes = [dense, vp, i64, vp]
        L.d3s_dense_workspace_bytes.argtypes = [dense]
        slopes = [vp, i64, vp, i64, i64, i64, i32, vp, i64, vp]
        L.d3s_dense_activation_backward_bf16.argtypes = slopes + [vp]
        L.d3s_dense_activation_backward_bf16_ws.argtypes = slopes + [vp, i64, vp]
        L.d3s_dense_activation_backward_workspace_bytes.argtypes = [i64, i64, i32]
        clip = [vp, vp, vp, vp, i32, f32, vp]
        L.d3s_clip_grads.argtypes = clip + [vp]
        L.d3s_clip_grads_ws.argtypes = clip + [vp, i64, vp]
        L.d3s_clip_grads_workspace_bytes.argtypes = [i32]
        for f in (L.d3s_logprob, L.d3s_logprob_ws, L.d3s_logprob_backward, L.d3s_dense_bf16, L.d3s_dense_bf16_ws,
                  L.d3s_dense_activation_backward_bf16, L.d3s_dense_activation_backward_bf16_ws, L.d3s_clip_grads,
                  L.d3s_clip_grads_ws):
            f.restype = i32
        for f in (L.d3s_logprob_workspace_bytes, L.d3s_dense_workspace_bytes,
                  L.d3s_dense_activation_backward_workspace_bytes, L.d3s_clip_grads_workspace_bytes):
            f.restype = i64
        verify = ctypes.POINTER(VerifyParams)
        u64 = ctypes.c_uint64
        L.d3s_verify.argtypes = [verify, vp]
        L.d3s_verify_ws.argtypes = [verify, vp, i64, vp]
        L.d3s_verify_workspace_bytes.argtypes = [verify]
        L.d3s_verify_ranked.argtypes = [vp, vp, i32, vp, vp, i32, i64, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp]
        L.d3s_embed.argtypes = [vp, i64, i32, vp, i32, i64, i64, i64, i64, f32, vp, i32, i64, vp]
        embed = [vp, i64, i32, vp, i32, i64, i64, i64, i64, f32, i32, vp, i32, i64]
        L.d3s_embed_backward.argtypes = embed + [vp]
        L.d3s_embed_backward_ws.argtypes = embed + [vp, i64, vp]
        L.d3s_embed_backward_workspace_bytes.argtypes = [i64, i32, i64, i64, i64]
        L.d3s_rms_norm.argtypes = [vp, i32, i64, vp, i64, vp, i64, vp, f32, i64, i64, vp, i32, i64, i32, vp, vp, vp]
        norm = [vp, i32, i64, vp, i64, vp, vp, vp, i64, i64, i64, vp, i64, vp]
        L.d3s_rms_norm_backward.argtypes = norm + [vp]
        L.d3s_rms_norm_backward_ws.argtypes = norm + [vp, i64, vp]
        L.d3s_rms_norm_backward_workspace_bytes.argtypes = [i64, i64, i32]
        L.d3s_dropout.argtypes = [vp, i32, i64, vp, i64, i64, i64, f32, u64, u64, vp, vp, i64, vp]
        for f in (L.d3s_verify, L.d3s_verify_ws, L.d3s_verify_ranked, L.d3s_embed, L.d3s_embed_backward,
                  L.d3s_embed_backward_ws, L.d3s_rms_norm, L.d3s_rms_norm_backward, L.d3s_rms_norm_backward_ws,
                  L.d3s_dropout):
            f.restype = i32
        for f in (L.d3s_verify_workspace_bytes, L.d3s_embed_backward_workspace_bytes,
                  L.d3s_rms_norm_backward_workspace_bytes):
            f.restype = i64
        L.d3s_version.argtypes = []
        L.d3s_version.restype = ctypes.c_char_p
        L.d3_sample.argtypes = [vp, i32, i32, f32, i32, f32, ctypes.c_ulonglong, vp]
        L.d3_sample.restype = None
        L.d3_sample_with_noise.argtypes = [vp, vp, i32, i32, i32, f32, f32, vp]
        L.d3_sample_with_noise.restype = None
        _lib = L
    return _lib


def sample_raw(logits, dtype, n_rows, vocab, row_stride, u, k, temperature, top_p, banned, ids,
               probs=None, cand=None, counters=None, flags=0, stream=None, noalloc=False, workspace=None):
    """d3s_sample (or d3s_sample_noalloc, or d3s_sample_ws with workspace =
    (address, bytes)) on device pointers (ints).  temperature / top_p: a
    float (scalar) or a device pointer wrapped as ("ptr", address)."""
    t_ptr, t_s = (temperature[1], 0.0) if isinstance(temperature, tuple) else (None, float(temperature))
    p_ptr, p_s = (top_p[1], 0.0) if isinstance(top_p, tuple) else (None, float(top_p))
    if workspace is not None:
        return lib().d3s_sample_ws(logits, dtype, n_rows, vocab, row_stride, u, k, t_ptr, p_ptr, t_s, p_s,
                                   banned, ids, probs, cand, counters, flags, workspace[0], workspace[1], stream)
    fn = lib().d3s_sample_noalloc if noalloc else lib().d3s_sample
    return fn(logits, dtype, n_rows, vocab, row_stride, u, k, t_ptr, p_ptr, t_s, p_s,
              banned, ids, probs, cand, counters, flags, stream)


def sample_seeded_raw(logits, dtype, n_rows, vocab, row_stride, seed, draw, k, temperature, top_p, banned, ids,
                      probs=None, cand=None, counters=None, flags=0, stream=None):
    """d3s_sample_seeded on device pointers (ints): the uniforms drawn in the
    kernel from (seed, draw), as d3s_uniform_fill would write them.
    temperature / top_p as in sample_raw."""
    t_ptr, t_s = (temperature[1], 0.0) if isinstance(temperature, tuple) else (None, float(temperature))
    p_ptr, p_s = (top_p[1], 0.0) if isinstance(top_p, tuple) else (None, float(top_p))
    return lib().d3s_sample_seeded(logits, dtype, n_rows, vocab, row_stride, seed, draw, k, t_ptr, p_ptr, t_s,
                                   p_s, banned, ids, probs, cand, counters, flags, stream)


def workspace_bytes(dtype, n_rows, vocab, k, flags=0):
    """d3s_sample_workspace_bytes: the workspace d3s_sample_ws needs (or a
    negative status)."""
    return lib().d3s_sample_workspace_bytes(dtype, n_rows, vocab, k, flags)


class Workspace:
    """A caller-owned workspace for the *_ws entry points: device memory of
    `nbytes`, cleared once by d3s_workspace_init on `stream`."""

    def __init__(self, nbytes, stream=None):
        import hiprt
        self.nbytes = max(int(nbytes), 256)
        self.buf = hiprt.DeviceBuffer(self.nbytes)
        rc = lib().d3s_workspace_init(self.buf.ptr, self.nbytes, stream.ptr if stream else None)
        if rc != OK:
            raise RuntimeError(f"d3s_workspace_init: {rc}")

    def arg(self):
        return (self.buf.ptr, self.nbytes)

    def free(self):
        self.buf.free()


def sample(logits, u, temperature, top_p, banned=None, flags=0, want_probs=True, row_stride=None,
           vocab=None, stream=None, noalloc=False, workspace=None, seed_draw=None):
    """Host arrays in, host arrays out (copies through device memory).
    logits: float32 or uint16 (bf16 bits) [N, row_stride]; u: float32 [N, k];
    temperature / top_p: scalars or float32 [N].  seed_draw = (seed, draw):
    d3s_sample_seeded instead, u then an int, k.  Returns dict(ids, probs,
    cand, counters, rc)."""
    import hiprt
    logits = np.ascontiguousarray(logits)
    dtype = DTYPE_F32 if logits.dtype == np.float32 else DTYPE_BF16
    if logits.dtype not in (np.float32, np.uint16):
        raise TypeError("logits must be float32 or uint16 (bf16 bits)")
    N = logits.shape[0]
    stride = logits.shape[1] if row_stride is None else row_stride
    V = stride if vocab is None else vocab
    bufs = dict(logits=hiprt.to_device(logits), ids=hiprt.DeviceBuffer(4 * N),
                counters=hiprt.DeviceBuffer(4 * NUM_COUNTERS).zero())
    if seed_draw is None:
        u = np.ascontiguousarray(u, np.float32)
        k = u.shape[1]
        bufs["u"] = hiprt.to_device(u)
    else:
        k = int(u)
    if want_probs:
        bufs["probs"] = hiprt.DeviceBuffer(4 * N * k)
        bufs["cand"] = hiprt.DeviceBuffer(4 * N * k)
    T = float(temperature) if not np.ndim(temperature) else None
    if np.ndim(temperature):
        bufs["Tbuf"] = hiprt.to_device(np.asarray(temperature, np.float32))
        T = ("ptr", bufs["Tbuf"].ptr)
    P = float(top_p) if not np.ndim(top_p) else None
    if np.ndim(top_p):
        bufs["Pbuf"] = hiprt.to_device(np.asarray(top_p, np.float32))
        P = ("ptr", bufs["Pbuf"].ptr)
    ban = None
    if banned is not None:
        bufs["ban"] = hiprt.to_device(np.asarray(banned, np.int32))
        ban = bufs["ban"].ptr
    if seed_draw is not None:
        rc = sample_seeded_raw(bufs["logits"].ptr, dtype, N, V, stride, seed_draw[0], seed_draw[1], k, T, P,
                               ban, bufs["ids"].ptr, bufs["probs"].ptr if want_probs else None,
                               bufs["cand"].ptr if want_probs else None, bufs["counters"].ptr, flags,
                               stream.ptr if stream else None)
    else:
        rc = sample_raw(bufs["logits"].ptr, dtype, N, V, stride, bufs["u"].ptr, k, T, P, ban,
                        bufs["ids"].ptr, bufs["probs"].ptr if want_probs else None,
                        bufs["cand"].ptr if want_probs else None, bufs["counters"].ptr, flags,
                        stream.ptr if stream else None, noalloc=noalloc,
                        workspace=workspace.arg() if isinstance(workspace, Workspace) else workspace)
    out = dict(rc=rc)
    if rc != OK:
        return out
    hiprt.synchronize()
    out["ids"] = bufs["ids"].download((N,), np.int32)
    out["counters"] = bufs["counters"].download((NUM_COUNTERS,), np.uint32)
    if want_probs:
        out["probs"] = bufs["probs"].download((N, k), np.float32)
        out["cand"] = bufs["cand"].download((N, k), np.int32)
    for b in bufs.values():
        if isinstance(b, hiprt.DeviceBuffer):
            b.free()
    return out


def uniform_fill(n, seed, draw):
    import hiprt
    buf = hiprt.DeviceBuffer(4 * n)
    rc = lib().d3s_uniform_fill(buf.ptr, n, seed, draw, None)
    if rc != OK:
        raise RuntimeError(f"d3s_uniform_fill: {rc}")
    hiprt.synchronize()
    return buf.download((n,), np.float32)


def math_selftest(x, divisor):
    import hiprt
    x = np.ascontiguousarray(x, np.float32)
    n = x.size
    bi = hiprt.to_device(x)
    be, bl, bd, bf = (hiprt.DeviceBuffer(4 * n), hiprt.DeviceBuffer(4 * n), hiprt.DeviceBuffer(4 * n),
                      hiprt.DeviceBuffer(8 * n))
    rc = lib().d3s_math_selftest(bi.ptr, be.ptr, bl.ptr, bd.ptr, bf.ptr, n, divisor, None)
    if rc != OK:
        raise RuntimeError(f"d3s_math_selftest: {rc}")
    hiprt.synchronize()
    return (be.download((n,), np.float32), bl.download((n,), np.float32),
            bd.download((n,), np.float32), bf.download((n,), np.uint64))


def exp2_selftest(x):
    """The hardware 2^x (v_exp_f32) behind the wave kernel's fast row sum."""
    import hiprt
    x = np.ascontiguousarray(x, np.float32)
    bi, bo = hiprt.to_device(x), hiprt.DeviceBuffer(4 * x.size)
    rc = lib().d3s_exp2_selftest(bi.ptr, bo.ptr, x.size, None)
    if rc != OK:
        raise RuntimeError(f"d3s_exp2_selftest: {rc}")
    hiprt.synchronize()
    return bo.download((x.size,), np.float32)


def log2_selftest(x):
    """The hardware log2 x (v_log_f32) behind the wave kernel's fast row sum's log."""
    import hiprt
    x = np.ascontiguousarray(x, np.float32)
    bi, bo = hiprt.to_device(x), hiprt.DeviceBuffer(4 * x.size)
    rc = lib().d3s_log2_selftest(bi.ptr, bo.ptr, x.size, None)
    if rc != OK:
        raise RuntimeError(f"d3s_log2_selftest: {rc}")
    hiprt.synchronize()
    return bo.download((x.size,), np.float32)


def d3_sample(logits, temperature, top_k, top_p, seed):
    """The reference's test export (src/testapi.c:155-166): host fp32 logits,
    a seed, host ids."""
    logits = np.ascontiguousarray(logits, np.float32)
    out = np.zeros(len(logits), np.int32)
    lib().d3_sample(logits.ctypes.data, logits.shape[0], logits.shape[1], temperature, top_k, top_p,
                    seed, out.ctypes.data)
    return out


def d3_sample_with_noise(logits, u, temperature, top_p):
    logits = np.ascontiguousarray(logits, np.float32)
    u = np.ascontiguousarray(u, np.float32)
    out = np.zeros(len(logits), np.int32)
    lib().d3_sample_with_noise(logits.ctypes.data, u.ctypes.data, logits.shape[0], logits.shape[1],
                               u.shape[1], temperature, top_p, out.ctypes.data)
    return out


def sample_ras_raw(logits, dtype, n_rows, vocab, row_stride, u, u_retry, history, history_len,
                   params, main_tok, code0=None, first_idx=None, retry_idx=None, counters=None,
                   stream=None):
    """d3s_sample_ras on device pointers (ints); params: RasParams."""
    return lib().d3s_sample_ras(logits, dtype, n_rows, vocab, row_stride, u, u_retry, history,
                                history_len, ctypes.byref(params) if params is not None else None,
                                main_tok, code0, first_idx, retry_idx, counters, stream)


def sample_ras(logits, u, u_retry, params, history=None, indices=True):
    """Host arrays in and out: logits float32 or uint16 (bf16 bits) [N, V];
    u [N, k], u_retry [N, k2]; history int32 [N, H] or None; params: dict of
    d3s_ras_params' fields; indices: ask for the two draws' indices too.
    Returns dict(rc, main, code0, first, retry, counters) (first / retry
    only with indices)."""
    import hiprt
    logits = np.ascontiguousarray(logits)
    dtype = DTYPE_F32 if logits.dtype == np.float32 else DTYPE_BF16
    N, V = logits.shape
    P = ras_params(**params)
    bufs = dict(logits=hiprt.to_device(logits), u=hiprt.to_device(np.ascontiguousarray(u, np.float32)),
                u2=hiprt.to_device(np.ascontiguousarray(u_retry, np.float32)),
                main=hiprt.DeviceBuffer(4 * N), code0=hiprt.DeviceBuffer(4 * N),
                first=hiprt.DeviceBuffer(4 * N), retry=hiprt.DeviceBuffer(4 * N),
                counters=hiprt.DeviceBuffer(4 * NUM_COUNTERS).zero())
    H = 0
    hist = None
    if history is not None and np.size(history):
        history = np.ascontiguousarray(history, np.int32).reshape(N, -1)
        H = history.shape[1]
        bufs["hist"] = hiprt.to_device(history)
        hist = bufs["hist"].ptr
    rc = sample_ras_raw(bufs["logits"].ptr, dtype, N, V, V, bufs["u"].ptr, bufs["u2"].ptr, hist, H, P,
                        bufs["main"].ptr, bufs["code0"].ptr, bufs["first"].ptr if indices else None,
                        bufs["retry"].ptr if indices else None, bufs["counters"].ptr)
    out = dict(rc=rc)
    if rc == OK:
        hiprt.synchronize()
        for name in ("main", "code0", "first", "retry") if indices else ("main", "code0"):
            out[name] = bufs[name].download((N,), np.int32)
        out["counters"] = bufs["counters"].download((NUM_COUNTERS,), np.uint32)
    for b in bufs.values():
        b.free()
    return out


def linear_bf16(x, w):
    """Host helper: x uint16 [N, K], w uint16 [V, K] (bf16 bits) -> uint16 [N, V]."""
    import hiprt
    x = np.ascontiguousarray(x, np.uint16)
    w = np.ascontiguousarray(w, np.uint16)
    N, K = x.shape
    V = w.shape[0]
    bx, bw, by = hiprt.to_device(x), hiprt.to_device(w), hiprt.DeviceBuffer(2 * N * V)
    rc = lib().d3s_linear_bf16(bx.ptr, bw.ptr, N, K, V, by.ptr, None)
    out = None
    if rc == OK:
        hiprt.synchronize()
        out = by.download((N, V), np.uint16)
    for b in (bx, bw, by):
        b.free()
    return rc, out



def linear_sample_bf16(x, w, u, temperature, top_p, flags=0, want_probs=True, keep_logits=True, stream=None):
    """Host helper for d3s_linear_sample_bf16: x uint16 [N, K], w uint16 [V, K]
    (bf16 bits), u float32 [N, k]; temperature / top_p scalars or float32 [N].
    Returns dict(rc, ids, probs, cand, counters, y) (y: the logits, uint16
    [N, V], when keep_logits)."""
    import hiprt
    x = np.ascontiguousarray(x, np.uint16)
    w = np.ascontiguousarray(w, np.uint16)
    u = np.ascontiguousarray(u, np.float32)
    N, K = x.shape
    V = w.shape[0]
    k = u.shape[1]
    bufs = dict(x=hiprt.to_device(x), w=hiprt.to_device(w), u=hiprt.to_device(u), ids=hiprt.DeviceBuffer(4 * N),
                counters=hiprt.DeviceBuffer(4 * NUM_COUNTERS).zero())
    if keep_logits:
        bufs["y"] = hiprt.DeviceBuffer(2 * N * V)
    if want_probs:
        bufs["probs"] = hiprt.DeviceBuffer(4 * N * k)
        bufs["cand"] = hiprt.DeviceBuffer(4 * N * k)
    t_ptr, t_s, p_ptr, p_s = None, 0.0, None, 0.0
    if np.ndim(temperature):
        bufs["T"] = hiprt.to_device(np.asarray(temperature, np.float32))
        t_ptr = bufs["T"].ptr
    else:
        t_s = float(temperature)
    if np.ndim(top_p):
        bufs["P"] = hiprt.to_device(np.asarray(top_p, np.float32))
        p_ptr = bufs["P"].ptr
    else:
        p_s = float(top_p)
    g = lambda name: bufs[name].ptr if name in bufs else None
    rc = lib().d3s_linear_sample_bf16(g("x"), g("w"), N, K, V, g("y"), g("u"), k, t_ptr, p_ptr, t_s, p_s,
                                      g("ids"), g("probs"), g("cand"), g("counters"), flags,
                                      stream.ptr if stream else None)
    out = dict(rc=rc)
    if rc == OK:
        hiprt.synchronize()
        out["ids"] = bufs["ids"].download((N,), np.int32)
        out["counters"] = bufs["counters"].download((NUM_COUNTERS,), np.uint32)
        if keep_logits:
            out["y"] = bufs["y"].download((N, V), np.uint16)
        if want_probs:
            out["probs"] = bufs["probs"].download((N, k), np.float32)
            out["cand"] = bufs["cand"].download((N, k), np.int32)
    for b in bufs.values():
        b.free()
    return out


# ---- scoring and training (include/d3s_train.h), on device pointers (ints) ----
def _temperature(temperature):
    return (temperature[1], 0.0) if isinstance(temperature, tuple) else (None, temperature)


def logprob_raw(logits, dtype, n_rows, vocab, row_stride, temperature, banned, tokens, n_tokens, logprobs,
                entropy=None, row_stats=None, n_top=0, top_ids=None, top_logprobs=None, counters=None, stream=None,
                workspace=None):
    """d3s_logprob, or d3s_logprob_ws with workspace = (address, bytes).
    temperature: a float, or a device pointer as ("ptr", address)."""
    t_ptr, t_s = _temperature(temperature)
    args = (logits, dtype, n_rows, vocab, row_stride, t_ptr, t_s, banned, tokens, n_tokens, logprobs, entropy,
            row_stats, n_top, top_ids, top_logprobs, counters)
    if workspace is not None:
        return lib().d3s_logprob_ws(*args, workspace[0], workspace[1], stream)
    return lib().d3s_logprob(*args, stream)


def logprob_backward_raw(logits, dtype, n_rows, vocab, row_stride, temperature, banned, tokens, n_tokens, row_stats,
                         entropy, grad_logprobs, grad_entropy, grad_logits, grad_row_stride, stream=None):
    """d3s_logprob_backward; temperature as in logprob_raw."""
    t_ptr, t_s = _temperature(temperature)
    return lib().d3s_logprob_backward(logits, dtype, n_rows, vocab, row_stride, t_ptr, t_s, banned, tokens, n_tokens,
                                      row_stats, entropy, grad_logprobs, grad_entropy, grad_logits, grad_row_stride,
                                      stream)


def dense_params(x, x_stride, w, w_stride, m, n, k, y, y_stride, y_dtype, x_transposed=False, w_transposed=False,
                 bias=None, activation=0, residual=None, residual_stride=0, z=None, z_stride=0):
    return DenseParams(x, x_stride, x_transposed, w, w_stride, w_transposed, m, n, k, bias, activation, residual,
                       residual_stride, z, z_stride, y, y_stride, y_dtype)


def dense_raw(x, x_stride, w, w_stride, m, n, k, y, y_stride, y_dtype, x_transposed=False, w_transposed=False,
              bias=None, activation=0, residual=None, residual_stride=0, z=None, z_stride=0, stream=None,
              workspace=None):
    """d3s_dense_bf16: y [m, n] = residual + act(x w^T + bias), or
    d3s_dense_bf16_ws with workspace = (address, bytes)."""
    p = DenseParams(x, x_stride, x_transposed, w, w_stride, w_transposed, m, n, k, bias, activation, residual,
                    residual_stride, z, z_stride, y, y_stride, y_dtype)
    if workspace is not None:
        return lib().d3s_dense_bf16_ws(ctypes.byref(p), workspace[0], workspace[1], stream)
    return lib().d3s_dense_bf16(ctypes.byref(p), stream)


def dense_activation_backward_raw(dy, dy_stride, z, z_stride, m, n, activation, dz, dz_stride, dbias, stream=None,
                                  workspace=None):
    """d3s_dense_activation_backward_bf16, or its _ws form with workspace =
    (address, bytes)."""
    args = (dy, dy_stride, z, z_stride, m, n, activation, dz, dz_stride, dbias)
    if workspace is not None:
        return lib().d3s_dense_activation_backward_bf16_ws(*args, workspace[0], workspace[1], stream)
    return lib().d3s_dense_activation_backward_bf16(*args, stream)


def clip_grads_raw(src, dst, numel, dtypes, n_tensors, max_norm, norm, stream=None, workspace=None):
    """d3s_clip_grads, or its _ws form with workspace = (address, bytes).  src,
    dst, numel, dtypes: host arrays' addresses (uint64, uint64 or None, int64,
    int32 per tensor)."""
    args = (src, dst, numel, dtypes, n_tensors, max_norm, norm)
    if workspace is not None:
        return lib().d3s_clip_grads_ws(*args, workspace[0], workspace[1], stream)
    return lib().d3s_clip_grads(*args, stream)


# ---- between ids and logits (include/d3s_step.h), on device pointers (ints) ----
def verify_params(target, target_dtype, target_stride, draft, draft_dtype, draft_stride, n_seqs, n_draft, vocab, drafted,
                  lengths, temperature, draft_temperature, u_accept, u_draw, tokens, n_accepted, accept=None,
                  counters=None):
    """VerifyParams; temperatures as in logprob_raw."""
    t_ptr, t_s = _temperature(temperature)
    d_ptr, d_s = _temperature(draft_temperature)
    return VerifyParams(target, target_dtype, target_stride, draft, draft_dtype, draft_stride, n_seqs, n_draft, vocab,
                        drafted, lengths, t_ptr, t_s, d_ptr, d_s, u_accept, u_draw, tokens, n_accepted, accept, counters)


def verify_raw(*args, stream=None, workspace=None, **kw):
    """d3s_verify, or d3s_verify_ws with workspace = (address, bytes); the other
    arguments are verify_params'."""
    p = verify_params(*args, **kw)
    if workspace is not None:
        return lib().d3s_verify_ws(ctypes.byref(p), workspace[0], workspace[1], stream)
    return lib().d3s_verify(ctypes.byref(p), stream)


def verify_ranked_raw(target_cand, target_probs, target_k, draft_cand, draft_probs, draft_k, n_seqs, n_draft, drafted,
                      lengths, u_accept, u_draw, tokens, n_accepted, accept=None, counters=None, stream=None):
    """d3s_verify_ranked."""
    return lib().d3s_verify_ranked(target_cand, target_probs, target_k, draft_cand, draft_probs, draft_k, n_seqs, n_draft,
                                   drafted, lengths, u_accept, u_draw, tokens, n_accepted, accept, counters, stream)


def embed_raw(ids, n_rows, n_ids, table, dtype, table_stride, vocab, slot_rows, width, scale, y, y_dtype, y_stride,
              stream=None):
    """d3s_embed: y[r] = scale * the sum of the ids' rows of the table."""
    return lib().d3s_embed(ids, n_rows, n_ids, table, dtype, table_stride, vocab, slot_rows, width, scale, y, y_dtype,
                           y_stride, stream)


def embed_backward_raw(ids, n_rows, n_ids, dy, dtype, dy_stride, vocab, slot_rows, width, scale, accumulate, grad,
                       grad_dtype, grad_stride, stream=None, workspace=None):
    """d3s_embed_backward, or its _ws form with workspace = (address, bytes)."""
    args = (ids, n_rows, n_ids, dy, dtype, dy_stride, vocab, slot_rows, width, scale, accumulate, grad, grad_dtype,
            grad_stride)
    if workspace is not None:
        return lib().d3s_embed_backward_ws(*args, workspace[0], workspace[1], stream)
    return lib().d3s_embed_backward(*args, stream)


def rms_norm_raw(x, dtype, x_stride, residual, residual_stride, sum, sum_stride, gain, eps, n_rows, width, y, y_dtype,
                 y_stride, group=0, scales=None, rstd=None, stream=None):
    """d3s_rms_norm."""
    return lib().d3s_rms_norm(x, dtype, x_stride, residual, residual_stride, sum, sum_stride, gain, eps, n_rows, width, y,
                              y_dtype, y_stride, group, scales, rstd, stream)


def rms_norm_backward_raw(dy, dtype, dy_stride, h, h_stride, gain, rstd, dsum, dsum_stride, n_rows, width, dx, dx_stride,
                          dgain, stream=None, workspace=None):
    """d3s_rms_norm_backward, or its _ws form with workspace = (address, bytes)."""
    args = (dy, dtype, dy_stride, h, h_stride, gain, rstd, dsum, dsum_stride, n_rows, width, dx, dx_stride, dgain)
    if workspace is not None:
        return lib().d3s_rms_norm_backward_ws(*args, workspace[0], workspace[1], stream)
    return lib().d3s_rms_norm_backward(*args, stream)


def dropout_raw(x, dtype, x_stride, residual, residual_stride, n_rows, width, p, seed, draw, draw_add, y, y_stride,
                stream=None):
    """d3s_dropout; its own gradient with x = dy and no residual."""
    return lib().d3s_dropout(x, dtype, x_stride, residual, residual_stride, n_rows, width, p, seed, draw, draw_add, y,
                             y_stride, stream)
