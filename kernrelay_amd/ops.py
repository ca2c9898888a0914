"""Op-level bindings of libkernrelay.so (include/kr_ops.h) for torch tensors.

torch only supplies device memory and the current stream; every op runs a
hand-written HIP kernel from the library. Calling an op with a CPU tensor or
without the built library raises: there is no CPU fallback.
"""

import ctypes
from array import array

from . import libapi

KR_BF16, KR_F16, KR_F32 = 0, 1, 2
EW = {"gelu": 0, "silu": 1, "cast": 2, "mul": 3, "add": 4, "swiglu": 5, "swiglu_gu": 6}
ROW = {"softmax": 0, "rmsnorm": 1, "add_rmsnorm": 2, "layernorm": 3}
CTRL_WORDS = 8


class KrWait(ctypes.Structure):
    _fields_ = [("ctrl", ctypes.c_void_p), ("flag0", ctypes.c_int32),
                ("state0", ctypes.c_int32), ("prod_rows", ctypes.c_int32),
                ("row_off", ctypes.c_int32), ("adv_lo", ctypes.c_int32),
                ("adv_hi", ctypes.c_int32), ("max_spins", ctypes.c_uint32)]


class KrPub(ctypes.Structure):
    _fields_ = [("ctrl", ctypes.c_void_p), ("flag0", ctypes.c_int32),
                ("rows_per_tile", ctypes.c_int32), ("arrivals", ctypes.c_int32)]


class KrCache(ctypes.Structure):
    """A paged key/value cache (kr_cache); make_cache fills it."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("layer_stride", ctypes.c_int64),
                ("page_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("layers", ctypes.c_int32), ("pages", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class KrSeqs(ctypes.Structure):
    """A launch's sequences (kr_seqs); make_seqs fills it."""
    _fields_ = [("table", ctypes.c_void_p), ("ld_table", ctypes.c_int64), ("lens", ctypes.c_void_p),
                ("starts", ctypes.c_void_p), ("tree", ctypes.c_void_p), ("ld_tree", ctypes.c_int64),
                ("table_pages", ctypes.c_int32), ("seqs", ctypes.c_int32),
                ("max_new", ctypes.c_int32), ("tree_words", ctypes.c_int32)]


class KrWeights(ctypes.Structure):
    """Attention weight per cached token (kr_weights); make_weights fills it."""
    _fields_ = [("w", ctypes.c_void_p), ("layer_stride", ctypes.c_int64), ("entry_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("layers", ctypes.c_int32), ("entries", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("width", ctypes.c_int32), ("entry", ctypes.c_void_p)]


class KrDrafts(ctypes.Structure):
    """Drafts and the target's logits (kr_drafts)."""
    _fields_ = [("logits", ctypes.c_void_p), ("ld_logits", ctypes.c_int64), ("draft", ctypes.c_void_p),
                ("ld_draft", ctypes.c_int64), ("tokens", ctypes.c_void_p), ("parents", ctypes.c_void_p),
                ("u", ctypes.c_void_p), ("u_next", ctypes.c_void_p), ("temperature", ctypes.c_void_p),
                ("dtype", ctypes.c_int32), ("draft_dtype", ctypes.c_int32), ("vocab", ctypes.c_int32),
                ("rows", ctypes.c_int32)]


class KrRope(ctypes.Structure):
    """Rotation tables and the gains of the per-head norms (kr_rope); make_rope fills it."""
    _fields_ = [("cos_t", ctypes.c_void_p), ("sin_t", ctypes.c_void_p), ("q_gamma", ctypes.c_void_p),
                ("k_gamma", ctypes.c_void_p), ("positions", ctypes.c_int64), ("head_dim", ctypes.c_int32),
                ("table_dtype", ctypes.c_int32), ("chain", ctypes.c_int32), ("eps", ctypes.c_float)]


_BOUND = False


def _lib():
    global _BOUND
    L = libapi.lib()
    if not _BOUND:
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        L.kr_ops_last_error.restype = ctypes.c_char_p
        L.kr_ops_last_error.argtypes = []
        L.kr_op_gemm.argtypes = [i32, vp, i64, vp, i64, vp, i64, vp, i32, i32, i32, i32,
                                 ctypes.POINTER(KrWait), ctypes.POINTER(KrPub), vp]
        L.kr_op_elementwise.argtypes = [i32, i32, i32, vp, vp, vp, i32, i32, i32, i32,
                                        ctypes.POINTER(KrWait), ctypes.POINTER(KrPub), vp]
        L.kr_op_rowop.argtypes = [i32, i32, vp, vp, vp, vp, vp, vp, i32, i32, f32, i32, i32,
                                  ctypes.POINTER(KrWait), ctypes.POINTER(KrPub), vp]
        L.kr_op_wait.argtypes = [ctypes.POINTER(KrWait), i32, i32, vp]
        L.kr_op_publish.argtypes = [ctypes.POINTER(KrPub), i32, vp]
        L.kr_op_embedding.argtypes = [vp, vp, vp, i32, i32, i64, vp]
        L.kr_op_rope.argtypes = [i32, vp, i64, i32, i32, i32, vp, vp, vp]
        L.kr_op_attention.argtypes = [i32, vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, f32, vp]
        L.kr_op_attention_workspace.argtypes = [i32, i32, i32, ctypes.POINTER(ctypes.c_size_t),
                                                ctypes.POINTER(ctypes.c_int)]
        L.kr_op_attention_split.argtypes = [i32, vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i32, i32, f32, vp,
                                            ctypes.c_size_t, vp, i32, vp]
        L.kr_op_transpose.argtypes = [vp, vp, i32, i32, vp]
        L.kr_op_gemm_swiglu.argtypes = [i32, vp, i64, vp, i64, vp, vp, i32, i32, i32, ctypes.POINTER(KrPub),
                                        i32, i32, vp]
        L.kr_op_gemm_swiglu_epilogue.argtypes = [i32, vp, i64, vp, i64, vp, i64, i32, i32, i32, vp]
        L.kr_op_gemm_streamk_workspace.argtypes = [i32, i32, i32, ctypes.POINTER(ctypes.c_size_t),
                                                    ctypes.POINTER(ctypes.c_int)]
        L.kr_op_gemm_streamk.argtypes = [i32, vp, i64, vp, i64, vp, i64, vp, i32, i32, i32, vp, ctypes.c_size_t, vp,
                                         i32, vp]
        L.kr_op_gemm_add_rmsnorm.argtypes = [i32, vp, i64, vp, i64, vp, i32, i32, i32, vp, vp, vp, vp, vp, f32,
                                             ctypes.POINTER(KrPub), ctypes.c_uint32, vp, ctypes.c_size_t, vp, i32, vp]
        L.kr_op_gemm_streamk_noalloc.argtypes = [i32, vp, i64, vp, i64, vp, i64, vp, i32, i32, i32, vp]
        sz, p = ctypes.c_size_t, ctypes.POINTER
        L.kr_op_qk_norm_rope.argtypes = [i32, p(KrRope), vp, i64, vp, i64, vp, i64, vp, i64, vp, i32, i32, i32, vp]
        L.kr_op_qk_norm_rope_cache.argtypes = [p(KrRope), p(KrCache), i32, vp, i64, vp, i64, vp, i64, vp, i64, vp, vp,
                                               i32, i32, vp]
        L.kr_op_attention_paged_workspace.argtypes = [p(KrCache), p(KrSeqs), i32, p(sz), p(ctypes.c_int)]
        L.kr_op_attention_paged.argtypes = [p(KrCache), i32, p(KrSeqs), vp, i64, vp, i64, i32, i32, f32, vp, sz, vp,
                                            i32, vp]
        L.kr_op_cache_copy_pages.argtypes = [p(KrCache), vp, vp, i32, vp]
        L.kr_op_cache_compact.argtypes = [p(KrCache), p(KrSeqs), vp, i64, i32, vp, vp]
        L.kr_op_attention_paged_lse.argtypes = [p(KrCache), i32, p(KrSeqs), vp, i64, vp, i64, vp, i64, i32, i32, f32,
                                                vp, sz, vp, i32, vp]
        L.kr_op_attention_paged_weigh_workspace.argtypes = [p(KrCache), p(KrSeqs), i32, p(sz)]
        L.kr_op_attention_paged_weigh.argtypes = [p(KrCache), i32, p(KrSeqs), vp, i64, vp, i64, i32, i32, f32,
                                                  p(KrWeights), i32, f32, vp, i64, i32, vp, vp, sz, vp]
        L.kr_op_cache_evict.argtypes = [p(KrCache), p(KrSeqs), p(KrWeights), i32, i32, i32, vp, vp]
        L.kr_op_verify_drafts_workspace.argtypes = [p(KrDrafts), p(KrSeqs), p(sz), p(ctypes.c_int)]
        L.kr_op_verify_drafts.argtypes = [p(KrDrafts), p(KrSeqs), vp, i64, i32, vp, vp, vp, sz, vp, i32, vp]
        L.kr_op_stream_create.argtypes = []
        L.kr_op_stream_create.restype = vp
        L.kr_op_stream_destroy.argtypes = [vp]
        L.kr_op_stream_destroy.restype = ctypes.c_int
        for name in ("kr_op_gemm", "kr_op_gemm_swiglu", "kr_op_gemm_swiglu_epilogue", "kr_op_gemm_streamk",
                     "kr_op_gemm_add_rmsnorm", "kr_op_gemm_streamk_noalloc",
                     "kr_op_gemm_streamk_workspace", "kr_op_elementwise", "kr_op_rowop", "kr_op_wait", "kr_op_publish",
                     "kr_op_embedding", "kr_op_rope", "kr_op_attention", "kr_op_attention_workspace",
                     "kr_op_attention_split", "kr_op_transpose", "kr_op_qk_norm_rope", "kr_op_qk_norm_rope_cache",
                     "kr_op_attention_paged_workspace", "kr_op_attention_paged", "kr_op_cache_copy_pages",
                     "kr_op_cache_compact", "kr_op_attention_paged_lse", "kr_op_attention_paged_weigh_workspace",
                     "kr_op_attention_paged_weigh", "kr_op_cache_evict", "kr_op_verify_drafts_workspace",
                     "kr_op_verify_drafts"):
            getattr(L, name).restype = ctypes.c_int
        _BOUND = True
    return L


# A launch's host side is Python for the most part, and the small kernels run
# in less time than it took (a gemm of a few rows: 5 us on the GPU, 8.5 per
# call): dtypes come from one table, addresses go to ctypes as plain ints, and
# the current stream's handle is read without making a torch Stream for it.
_DT = {}


def _dt(t):
    if not _DT:
        import torch
        _DT.update({torch.bfloat16: KR_BF16, torch.float16: KR_F16, torch.float32: KR_F32})
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError("unsupported dtype %s" % t.dtype) from None


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError("kernrelay ops need device tensors (got a CPU tensor)")
    return t.data_ptr()


_RAW = None  # (current device, current stream handle of a device)


def _stream(stream):
    if stream is not None:
        return stream.cuda_stream
    global _RAW
    if _RAW is None:
        import torch
        torch.cuda.current_stream()  # initialises the device as any torch call does
        get = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if get is None:  # a torch without the raw accessor
            _RAW = (int, lambda _: torch.cuda.current_stream().cuda_stream)
        else:
            _RAW = (torch._C._cuda_getDevice, get)
    return _RAW[1](_RAW[0]())


class QueueStream:
    """A stream on a hardware queue of its own (kr_op_stream_create): relay
    parties that wait on each other on the device need two of these. Usable
    wherever the op wrappers take a stream."""

    def __init__(self):
        h = _lib().kr_op_stream_create()
        if not h:
            raise RuntimeError("kr_op_stream_create failed: %s" % _lib().kr_ops_last_error().decode())
        self.cuda_stream = h

    def close(self):
        if self.cuda_stream:
            _check(_lib().kr_op_stream_destroy(ctypes.c_void_p(self.cuda_stream)))
            self.cuda_stream = None


def _check(rc):
    if rc != 0:
        raise RuntimeError("kernrelay op failed: %s" % _lib().kr_ops_last_error().decode())


def make_wait(ctrl, flag0, state0, prod_rows, row_off=0, adv=(0, 0), max_spins=0):
    return KrWait(ctypes.c_void_p(ctrl.data_ptr()), flag0, state0, prod_rows, row_off,
                  adv[0], adv[1], max_spins)


def make_pub(ctrl, flag0, rows_per_tile):
    return KrPub(ctypes.c_void_p(ctrl.data_ptr()), flag0, rows_per_tile, 0)


def gemm(A, Bt, C, bias=None, pub=None, bm=0, wait=None, stream=None):
    """C[M,N] = A[M,K] @ Bt[N,K]^T (+bias), bf16/f16 in and out. `wait`: each
    workgroup first waits for the relay tiles of A it reads."""
    M, K = A.shape
    N = Bt.shape[0]
    assert Bt.shape[1] == K and C.shape[0] == M and C.shape[1] == N
    _check(_lib().kr_op_gemm(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(C), C.stride(0),
                             _ptr(bias), M, N, K, bm, ctypes.byref(wait) if wait else None,
                             ctypes.byref(pub) if pub else None, _stream(stream)))


def gemm_swiglu(A, Bt, C, act, pub, tail_tiles=0, order_rows=0, stream=None):
    """C[M, 2I] = A @ Bt^T released in relay tiles (pub); act[M, I] =
    SwiGLU of C over the first tail_tiles relay tiles (0 = all) by workgroups
    appended to the same launch."""
    M, K = A.shape
    cols = act.shape[1]
    assert Bt.shape == (2 * cols, K) and C.shape == (M, 2 * cols) and act.shape[0] == M
    _check(_lib().kr_op_gemm_swiglu(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(C), _ptr(act),
                                    M, cols, K, ctypes.byref(pub), tail_tiles, order_rows, _stream(stream)))


def gemm_add_rmsnorm(A, Bt, C, res, gamma, y, pub, sum_out=None, rstd=None, eps=1e-6, ws=None, counters=None,
                     max_spins=0, stream=None):
    """C = A @ Bt^T released in relay tiles (pub); the launch's own
    workgroups compute Add+RMSNorm(res + C) of each released tile (y, sum_out,
    rstd), the bits of rowop("add_rmsnorm"). ws/counters: stream-K workspace
    (None: data-parallel)."""
    M, K = A.shape
    N = Bt.shape[0]
    assert Bt.shape[1] == K and C.shape == (M, N) and res.shape == (M, N) and y.shape == (M, N)
    # the C entry takes C, res, y and sum_out as packed [M, N] rows and rstd
    # as [M]: a strided view would be read or written with row stride N
    for name, t in (("C", C), ("res", res), ("y", y), ("sum_out", sum_out), ("rstd", rstd), ("gamma", gamma)):
        if t is not None and not t.is_contiguous():
            raise ValueError("gemm_add_rmsnorm: %s must be contiguous" % name)
    if sum_out is not None and sum_out.shape != (M, N):
        raise ValueError("gemm_add_rmsnorm: sum_out must be [M, N]")
    if rstd is not None and rstd.numel() != M:
        raise ValueError("gemm_add_rmsnorm: rstd must hold M values")
    _check(_lib().kr_op_gemm_add_rmsnorm(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(C), M, N, K,
                                         _ptr(res), _ptr(gamma), _ptr(y), _ptr(sum_out), _ptr(rstd), ctypes.c_float(eps),
                                         ctypes.byref(pub), ctypes.c_uint32(max_spins), _ptr(ws),
                                         0 if ws is None else ws.numel() * ws.element_size(), _ptr(counters),
                                         0 if counters is None else counters.numel(), _stream(stream)))


def gemm_streamk_workspace(M, N, K):
    """(workspace bytes, counters) a stream-K GEMM of this shape needs; (0, 0)
    when it runs data-parallel."""
    b, c = ctypes.c_size_t(0), ctypes.c_int(0)
    _check(_lib().kr_op_gemm_streamk_workspace(M, N, K, ctypes.byref(b), ctypes.byref(c)))
    return b.value, c.value


def gemm_streamk(A, Bt, C, ws, counters, bias=None, stream=None):
    """C = A @ Bt^T (+bias) split stream-K over the CUs (ws: uint8 device
    tensor, counters: int32 device tensor, zero before the first call)."""
    M, K = A.shape
    N = Bt.shape[0]
    _check(_lib().kr_op_gemm_streamk(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(C), C.stride(0),
                                     _ptr(bias), M, N, K, _ptr(ws), ws.numel() * ws.element_size(),
                                     _ptr(counters), counters.numel(), _stream(stream)))


def gemm_streamk_noalloc(A, Bt, C, bias=None, stream=None):
    """gemm_streamk with the library's own scratch (no workspace argument,
    nothing allocated); raises for a split larger than the scratch. Products
    with M or N below 256 or K below 2048 take none: as gemm."""
    M, K = A.shape
    N = Bt.shape[0]
    _check(_lib().kr_op_gemm_streamk_noalloc(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(C),
                                             C.stride(0), _ptr(bias), M, N, K, _stream(stream)))


def gemm_swiglu_epilogue(A, Bt, act, stream=None):
    """act[M, I] = SwiGLU of A @ Bt^T (Bt = [2I, K], gate/up interleaved in
    groups of 8 rows), applied in the GEMM's epilogue; the product itself is
    never written."""
    M, K = A.shape
    cols = act.shape[1]
    assert Bt.shape == (2 * cols, K) and act.shape[0] == M
    _check(_lib().kr_op_gemm_swiglu_epilogue(_dt(A), _ptr(A), A.stride(0), _ptr(Bt), Bt.stride(0), _ptr(act),
                                             act.stride(0), M, cols, K, _stream(stream)))


def elementwise(op, x0, y, x1=None, rows=None, cols=None, tile_rows=0, grid=0, wait=None, pub=None,
                stream=None):
    rows = rows if rows is not None else y.shape[0]
    cols = cols if cols is not None else y.shape[-1]
    _check(_lib().kr_op_elementwise(EW[op], _dt(x0), _dt(y), _ptr(x0), _ptr(x1), _ptr(y), rows, cols,
                                    tile_rows, grid, ctypes.byref(wait) if wait else None,
                                    ctypes.byref(pub) if pub else None, _stream(stream)))


def rowop(op, x0, y, x1=None, gamma=None, sum_out=None, rstd_out=None, eps=1e-6, tile_rows=0, grid=0,
          wait=None, pub=None, stream=None):
    rows, cols = y.shape
    _check(_lib().kr_op_rowop(ROW[op], _dt(x0), _ptr(x0), _ptr(x1), _ptr(gamma), _ptr(y), _ptr(sum_out),
                              _ptr(rstd_out), rows, cols, float(eps), tile_rows, grid,
                              ctypes.byref(wait) if wait else None, ctypes.byref(pub) if pub else None,
                              _stream(stream)))


def wait(w, lo, hi, stream=None):
    _check(_lib().kr_op_wait(ctypes.byref(w), lo, hi, _stream(stream)))


def publish(p, tile, stream=None):
    _check(_lib().kr_op_publish(ctypes.byref(p), tile, _stream(stream)))


def embedding(table, ids, out, stream=None):
    rows, cols = out.shape
    _check(_lib().kr_op_embedding(_ptr(table), _ptr(ids), _ptr(out), rows, cols, table.shape[0],
                                  _stream(stream)))


def rope(x, S, heads, D, cos_t, sin_t, ld=None, stream=None):
    _check(_lib().kr_op_rope(_dt(x), _ptr(x), ld if ld is not None else heads * D, S, heads, D,
                             _ptr(cos_t), _ptr(sin_t), _stream(stream)))


def attention(q, k, v, out, S, HQ, HKV, D, scale=None, ldq=0, ldk=0, ldv=0, ldo=0, stream=None):
    scale = scale if scale is not None else D ** -0.5
    _check(_lib().kr_op_attention(_dt(q), _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, _ptr(out), ldo,
                                  S, HQ, HKV, D, float(scale), _stream(stream)))


def attention_workspace(S, HQ, D):
    """(workspace bytes, counters) attention_split needs; (0, 0) when no query
    row is long enough to split."""
    b, c = ctypes.c_size_t(0), ctypes.c_int(0)
    _check(_lib().kr_op_attention_workspace(S, HQ, D, ctypes.byref(b), ctypes.byref(c)))
    return b.value, c.value


def attention_split(q, k, v, out, S, HQ, HKV, D, ws, counters, scale=None, ldq=0, ldk=0, ldv=0, ldo=0,
                    stream=None):
    scale = scale if scale is not None else D ** -0.5
    _check(_lib().kr_op_attention_split(_dt(q), _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv, _ptr(out), ldo,
                                        S, HQ, HKV, D, float(scale), _ptr(ws), ws.numel() * ws.element_size(),
                                        _ptr(counters), counters.numel(), _stream(stream)))


def transpose(src, dst, stream=None):
    R, C = src.shape
    assert dst.shape[0] == C and dst.shape[1] == R
    _check(_lib().kr_op_transpose(_ptr(src), _ptr(dst), R, C, _stream(stream)))


# ------------------------------------------------------------- paged cache
# Handles are made once and passed to every call (their tensors are kept
# alive with them); the calls check what the C entry cannot see: shapes,
# strides and devices of the tensors. The checks are one expression per tensor
# and the reason is looked for only after a refusal: the step kernels run in
# 3 to 7 us, and the wrappers' own time is what a caller of them waits for.
def _need(ok, who, what):
    if not ok:
        raise ValueError("%s: %s" % (who, what))


_INTS = None  # (torch.int32, torch.int64)


def _ints():
    global _INTS
    if _INTS is None:
        import torch
        _INTS = (torch.int32, torch.int64)
    return _INTS


def _heads(t, shape, dtype, who, name):
    """Address and row stride of a [rows, heads, D] tensor with packed heads."""
    s = t.stride()
    if t.dtype == dtype and t.shape == shape and s[2] == 1 and (s[1] == shape[2] or shape[1] == 1):
        if shape[0] <= 1:
            return t.data_ptr(), 0
        if s[0] >= shape[1] * shape[2]:
            return t.data_ptr(), s[0]
        raise ValueError("%s: %s: rows overlap" % (who, name))
    _need(t.shape == shape and t.dtype == dtype, who, "%s must be %s %s" % (name, tuple(shape), dtype))
    raise ValueError("%s: %s: the heads of a row must be packed" % (who, name))


def _vector(t, dtype, n, who, name):
    """Address of a contiguous [n] tensor."""
    if t.dtype == dtype and t.shape == (n,) and (n <= 1 or t.stride(0) == 1):
        return t.data_ptr()
    raise ValueError("%s: %s must be a contiguous %s vector of %d" % (who, name, dtype, n))


def _pitch(t, who, name):
    """Row stride of a [rows, n] tensor with contiguous rows."""
    rows, n = t.shape
    if rows <= 1:
        return n
    _need(t.stride(0) >= n, who, "%s: rows overlap" % name)
    return t.stride(0)


def _launch_stream(stream, who, dev, other, *tensors):
    """The stream's handle. Kernels go to the current device's streams: the
    handles' tensors and the call's must be on it."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            if not t.is_cuda:
                raise RuntimeError("kernrelay ops need device tensors (got a CPU tensor)")
            raise ValueError("%s: a tensor is on %s, the handle's are on device %d" % (who, t.device, dev))
    if _RAW is None:
        _stream(None)
    if dev != other or _RAW[0]() != dev:
        raise ValueError("%s: the handles' tensors are on devices %d and %d, the current device is %d" % (
            who, dev, other, _RAW[0]()))
    if stream is not None and getattr(stream, "device_index", dev) != dev:
        raise ValueError("%s: the stream is on device %d, the handles' tensors are on device %d" % (
            who, stream.device_index, dev))
    return _stream(stream)


def make_cache(k, v):
    """Handle of a paged cache: k and v [layers, pages, page_size, heads,
    head_dim] (or without layers), bf16 or f16, the same strides, rows of
    head_dim contiguous."""
    who = "make_cache"
    _need(k.shape == v.shape and k.dtype == v.dtype and k.stride() == v.stride(), who,
          "k and v must agree in shape, type and strides")
    _need(k.dim() in (4, 5), who, "k and v are [layers, pages, page_size, heads, head_dim]")
    _need(k.stride(-1) == 1, who, "rows must be contiguous")
    _need(k.device == v.device, who, "k and v must be on one device")
    shape, stride = list(k.shape), list(k.stride())
    if len(shape) == 4:
        shape, stride = [1] + shape, [0] + stride
    c = KrCache(_ptr(k), _ptr(v), *stride[:4], *shape, _dt(k))
    c.keep, c.device, c.torch_dtype = (k, v), k.get_device(), k.dtype
    return c


def check_tree(tree, max_new, who):
    """Words and row stride of make_seqs' tree; refuses one that is none."""
    _need(tree.dtype == _ints()[1] and tree.dim() == 2 and (tree.shape[1] <= 1 or tree.stride(1) == 1), who,
          "tree must be int64 [rows, words] with contiguous rows")
    words, ld = tree.shape[1], _pitch(tree, who, "tree")
    _need(max_new <= 64 * words, who, "the tree has too few words for max_new")
    return words, ld


def make_seqs(table, lens, starts, max_new, tree=None):
    """Handle of a launch's sequences: table [seqs, pages] and lens [seqs]
    int32, starts [seqs + 1] int32 (rows starts[b] .. starts[b + 1] - 1 are
    sequence b's new tokens), all read on the device at each call. max_new: no
    sequence has more new tokens. tree [rows, words] int64: bit j % 64 of word
    j // 64 says whether the row sees new token j of its sequence (None:
    causal)."""
    import torch
    who = "make_seqs"
    _need(table.dtype == torch.int32 and table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1), who,
          "table must be int32 [seqs, pages] with contiguous rows")
    n = table.shape[0]
    for v, size, name in ((lens, n, "lens"), (starts, n + 1, "starts")):
        _need(v.dtype == torch.int32 and v.shape == (size,) and v.is_contiguous(), who,
              "%s must be a contiguous int32 vector of %d" % (name, size))
    _need(0 <= max_new < 1 << 31, who, "max_new must not be negative, nor past 32 bits")
    ld_table = _pitch(table, who, "table")
    words, ld = (0, 0) if tree is None else check_tree(tree, max_new, who)
    tensors = [t for t in (table, lens, starts, tree) if t is not None]
    _need(len({t.device for t in tensors}) == 1, who, "the tensors must be on one device")
    s = KrSeqs(_ptr(table), ld_table, _ptr(lens), _ptr(starts), _ptr(tree), ld,
               table.shape[1], n, max_new, words)
    s.keep, s.device, s.rows = tensors, table.get_device(), None if tree is None else tree.shape[0]
    return s


def make_rope(cos_t, sin_t, q_gamma=None, k_gamma=None, eps=1e-6, chain=False):
    """Handle of rotation tables [positions, head_dim] (fp32 or the
    activations' type) and, optionally, the gains [head_dim] of the per-head
    norms of q and k. chain: round after each step, the bits of rowop
    ("rmsnorm") and rope in sequence; otherwise once, at the store."""
    who = "make_rope"
    _need(cos_t.dim() == 2 and cos_t.shape == sin_t.shape and cos_t.dtype == sin_t.dtype and cos_t.is_contiguous()
          and sin_t.is_contiguous(), who, "cos and sin must be contiguous [positions, head_dim] of one type")
    _need((q_gamma is None) == (k_gamma is None), who, "one of the two gains is missing")
    for g in (q_gamma, k_gamma):
        _need(g is None or (g.shape == cos_t.shape[1:] and g.is_contiguous() and g.dtype == q_gamma.dtype), who,
              "gains must be [head_dim] of one type")
    tensors = [t for t in (cos_t, sin_t, q_gamma, k_gamma) if t is not None]
    _need(len({t.device for t in tensors}) == 1, who, "the tensors must be on one device")
    r = KrRope(_ptr(cos_t), _ptr(sin_t), _ptr(q_gamma), _ptr(k_gamma), cos_t.shape[0], cos_t.shape[1], _dt(cos_t),
               int(bool(chain)), float(eps))
    r.keep, r.device = tensors, cos_t.get_device()
    r.torch_dtype = None if q_gamma is None else q_gamma.dtype
    return r


def qk_norm_rope(rope, q, k, q_out, k_out, positions=None, stream=None):
    """q_out, k_out = per-head RMSNorm (if the handle has gains) and rotation
    of q [rows, HQ, D] and k [rows, HKV, D] in one pass. Row r stands at
    positions[r] (int64; None: r); outside the tables: zeros. Outputs may be
    the inputs themselves; other overlaps are refused."""
    who = "qk_norm_rope"
    _need(q.dim() == 3 and k.dim() == 3, who, "q and k are [rows, heads, head_dim]")
    qs, ks, dt, dev = q.shape, k.shape, q.dtype, rope.device
    rows = qs[0]
    _need(qs[2] == rope.head_dim, who, "the tables have another head_dim")
    _need(rope.torch_dtype in (None, dt), who, "the gains must be of q's type")
    _need(ks[0] == rows and ks[2] == qs[2], who, "k must be [%d, heads, %d]" % (rows, qs[2]))
    qp, ldq = _heads(q, qs, dt, who, "q")
    kp, ldk = _heads(k, ks, dt, who, "k")
    qo, ldqo = _heads(q_out, qs, dt, who, "q_out")
    ko, ldko = _heads(k_out, ks, dt, who, "k_out")
    pos = None if positions is None else _vector(positions, _ints()[1], rows, who, "positions")
    _check(_lib().kr_op_qk_norm_rope(_dt(q), rope, qp, ldq, kp, ldk, qo, ldqo, ko, ldko, pos, rows, qs[1], ks[1],
                                     _launch_stream(stream, who, dev, dev, q, k, q_out, k_out, positions)))


def qk_norm_rope_cache(rope, cache, layer, q, k, v, q_out, positions, slots, stream=None):
    """qk_norm_rope with row r's k and v written to slot slots[r] (int64: page *
    page_size + row in the page; outside the cache, say -1: not written) of a
    layer of the cache. No two rows may share a slot."""
    who = "qk_norm_rope_cache"
    _need(q.dim() == 3, who, "q is [rows, heads, head_dim]")
    qs, dt, dev, i64 = q.shape, cache.torch_dtype, cache.device, _ints()[1]
    rows = qs[0]
    kv = (rows, cache.heads, cache.head_dim)
    _need(qs[2] == kv[2], who, "q has another head_dim than the cache")
    _need(rope.torch_dtype in (None, dt), who, "the gains must be of the cache's type")
    qp, ldq = _heads(q, qs, dt, who, "q")
    kp, ldk = _heads(k, kv, dt, who, "k")
    vp, ldv = _heads(v, kv, dt, who, "v")
    qo, ldqo = _heads(q_out, qs, dt, who, "q_out")
    pos = None if positions is None else _vector(positions, i64, rows, who, "positions")
    _check(_lib().kr_op_qk_norm_rope_cache(rope, cache, layer, qp, ldq, kp, ldk, vp, ldv, qo, ldqo, pos,
                                           _vector(slots, i64, rows, who, "slots"), rows, qs[1],
                                           _launch_stream(stream, who, dev, rope.device, q, k, v, q_out, positions,
                                                          slots)))


def attention_paged_workspace(cache, seqs, HQ):
    """(workspace bytes, counters) with which attention_paged cuts long
    sequences into pieces; (0, 0) when it never would."""
    b, c = ctypes.c_size_t(0), ctypes.c_int(0)
    _check(_lib().kr_op_attention_paged_workspace(cache, seqs, HQ, ctypes.byref(b), ctypes.byref(c)))
    return b.value, c.value


def attention_paged(cache, layer, seqs, q, out, scale=None, ws=None, counters=None, stream=None, lse=None):
    """Attention of a launch's new tokens q [rows, HQ, D] over a layer of the
    cache; their own keys and values are in the cache already, and out
    overlaps neither q nor the layer. ws (uint8) and counters (int32, zero before the
    first call): of attention_paged_workspace's sizes for these handles at
    least (a wider table or more sequences may need more), for one stream at a
    time; None: no sequence is cut into pieces. lse [rows, HQ] float32: gets
    the logarithms of the rows' sums, for attention_paged_weigh."""
    who = "attention_paged"
    _need(q.dim() == 3, who, "q is [rows, heads, head_dim]")
    shape, dt, dev = q.shape, cache.torch_dtype, cache.device
    _need(shape[2] == cache.head_dim, who, "q has another head_dim than the cache")
    _need(seqs.rows is None or seqs.rows >= shape[0], who, "the tree has too few rows")
    qp, ldq = _heads(q, shape, dt, who, "q")
    op, ldo = _heads(out, shape, dt, who, "out")
    wp, cp, nbytes, ncnt = None, None, 0, 0
    if ws is not None:
        _need(counters is not None and counters.dtype == _ints()[0] and counters.dim() == 1 and counters.is_contiguous()
              and ws.is_contiguous(), who, "ws and counters (an int32 vector) must be contiguous")
        # (an empty tensor's address is 0, which would say that there is none; at
        # 0 bytes no address is used, and too few are refused)
        wp, cp, nbytes, ncnt = ws.data_ptr() or 16, counters.data_ptr(), ws.nbytes, counters.shape[0]
    scale = cache.head_dim ** -0.5 if scale is None else scale
    if lse is not None:
        lp, ld_lse = _rows32(lse, shape, who, "lse")
        _check(_lib().kr_op_attention_paged_lse(cache, layer, seqs, qp, ldq, op, ldo, lp, ld_lse, shape[0], shape[1],
                                                scale, wp, nbytes, cp, ncnt,
                                                _launch_stream(stream, who, dev, seqs.device, q, out, ws, counters,
                                                               lse)))
        return
    _check(_lib().kr_op_attention_paged(cache, layer, seqs, qp, ldq, op, ldo, shape[0], shape[1], scale, wp, nbytes,
                                        cp, ncnt, _launch_stream(stream, who, dev, seqs.device, q, out, ws, counters)))


def _rows32(t, shape, who, name):
    """Address and row stride of a float32 [rows, heads] tensor, as q's shape has them."""
    if t.dtype == _f32() and t.shape == shape[:2] and (shape[1] == 1 or t.stride(1) == 1):
        return t.data_ptr(), _pitch(t, who, name)
    raise ValueError("%s: %s must be float32 %s with contiguous rows" % (who, name, tuple(shape[:2])))


_F32 = None


def _f32():
    global _F32
    if _F32 is None:
        import torch
        _F32 = torch.float32
    return _F32


def cache_copy_pages(cache, src, dst, stream=None):
    """Page dst[i] becomes a copy of page src[i] in every layer (lists of page
    ids, no page twice in dst and none in both)."""
    who = "cache_copy_pages"
    a, b = array("i", src), array("i", dst)
    _need(len(a) == len(b), who, "src and dst differ in length")
    _check(_lib().kr_op_cache_copy_pages(cache, a.buffer_info()[0], b.buffer_info()[0], len(a),
                                         _launch_stream(stream, who, cache.device, cache.device)))


def cache_compact(cache, seqs, path, path_lens, stream=None):
    """Accepted drafts move to the front: in every layer and for each sequence
    the rows at lens[b] + path[b, i], i < path_lens[b], go to lens[b] + i, as if
    all were read before any is written. path [seqs, width <= 256] and
    path_lens [seqs] int32; entries below 0 move nothing."""
    who = "cache_compact"
    n, dev, i32 = seqs.seqs, cache.device, _ints()[0]
    _need(path.dim() == 2 and path.dtype == i32 and path.shape[0] == n and (path.shape[1] <= 1 or path.stride(1) == 1),
          who, "path must be int32 [seqs, width] with contiguous rows")
    lens = _vector(path_lens, i32, n, who, "path_lens")
    width = path.shape[1]
    _check(_lib().kr_op_cache_compact(cache, seqs, path.data_ptr(), _pitch(path, who, "path"), width, lens,
                                      _launch_stream(stream, who, dev, seqs.device, path, path_lens)))


# ------------------------------------------------- after a step over the cache
def make_weights(w, entry=None):
    """Handle of the attention weight that cached tokens got: w float32
    [layers, entries, heads, width] (or without layers), rows of width
    contiguous and none overlapping. entry [seqs] int32, read on the device at
    each call: where in w a launch's sequence b stands (None: at b; outside w:
    nowhere, and the calls leave it alone). No two sequences of a launch may
    have the same entry."""
    who = "make_weights"
    _need(w.dim() in (3, 4) and w.dtype == _f32(), who, "w must be float32 [layers, entries, heads, width]")
    _need(w.shape[-1] <= 1 or w.stride(-1) == 1, who, "rows must be contiguous")
    _need(all(0 < n < 1 << 31 for n in w.shape), who, "w is empty, or too large")
    shape, stride = list(w.shape), list(w.stride())
    if len(shape) == 3:
        shape, stride = [1] + shape, [0] + stride
    if entry is not None:
        _need(entry.dtype == _ints()[0] and entry.dim() == 1 and (entry.shape[0] <= 1 or entry.stride(0) == 1), who,
              "entry must be a contiguous int32 vector")
        _need(entry.device == w.device, who, "w and entry must be on one device")
    h = KrWeights(_ptr(w), *stride[:3], *shape, _ptr(entry))
    h.keep, h.device, h.seqs = (w, entry), w.get_device(), None if entry is None else entry.shape[0]
    return h


def _of_weights(weights, cache, seqs, who):
    _need(weights.device == cache.device, who, "the weights are on another device than the cache")
    if weights.seqs is None:
        _need(weights.entries >= seqs.seqs, who, "the weights have fewer entries than there are sequences")
    else:
        _need(weights.seqs == seqs.seqs, who, "entry must name one entry for each sequence")


def attention_paged_weigh_workspace(cache, seqs, HQ):
    """Bytes of workspace that attention_paged_weigh needs for these handles."""
    b = ctypes.c_size_t(0)
    _check(_lib().kr_op_attention_paged_weigh_workspace(cache, seqs, HQ, ctypes.byref(b)))
    return b.value


def attention_paged_weigh(cache, layer, seqs, q, lse, weights, ws, scale=None, last=0, decay=1.0, path=None,
                          path_lens=None, stream=None):
    """Adds the attention weight that each cached token gets from a launch's new
    tokens q [rows, HQ, D] to its weight (make_weights) times `decay`, key head
    by key head; a new token's weight becomes what it gets. lse [rows, HQ]: of
    attention_paged for the same handles and scale. last > 0: only the last
    `last` new tokens of each sequence count. path [seqs, width], path_lens
    [seqs] int32: the drafts have been accepted and moved together by
    cache_compact with these; only their rows count. ws: uint8 of
    attention_paged_weigh_workspace's size, for one stream at a time."""
    who = "attention_paged_weigh"
    _need(q.dim() == 3, who, "q is [rows, heads, head_dim]")
    shape, dev, i32 = q.shape, cache.device, _ints()[0]
    _need(shape[2] == cache.head_dim, who, "q has another head_dim than the cache")
    _need(seqs.rows is None or path is not None or seqs.rows >= shape[0], who, "the tree has too few rows")
    _of_weights(weights, cache, seqs, who)
    qp, ldq = _heads(q, shape, cache.torch_dtype, who, "q")
    lp, ld_lse = _rows32(lse, shape, who, "lse")
    _need((path is None) == (path_lens is None), who, "a path needs its lengths")
    pp, ld_path, width, pl = None, 0, 0, None
    if path is not None:
        _need(path.dim() == 2 and path.dtype == i32 and path.shape[0] == seqs.seqs
              and (path.shape[1] <= 1 or path.stride(1) == 1), who, "path must be int32 [seqs, width] with contiguous rows")
        _need(path.shape[1] > 0 or seqs.seqs == 0, who, "path rows are empty")
        pl = _vector(path_lens, i32, seqs.seqs, who, "path_lens")
        pp, ld_path, width = path.data_ptr(), _pitch(path, who, "path"), path.shape[1]
    _need(ws.is_contiguous(), who, "ws must be contiguous")
    _check(_lib().kr_op_attention_paged_weigh(cache, layer, seqs, qp, ldq, lp, ld_lse, shape[0], shape[1],
                                              cache.head_dim ** -0.5 if scale is None else scale, weights, last, decay,
                                              pp, ld_path, width, pl, ws.data_ptr(), ws.nbytes,
                                              _launch_stream(stream, who, dev, seqs.device, q, lse, ws, path,
                                                             path_lens)))


def cache_evict(cache, seqs, weights, keep, sinks=0, recent=0, stream=None):
    """Sequences of more than budget = keep.shape[3] tokens come down to that
    many, layer by layer and key head by key head: the first `sinks`, the last
    `recent` and of the others those with the largest weights stay. keep [layers,
    seqs, heads, budget] int32 (packed) gets which token the one at each place
    was (-1 behind the last). What stands where it may stay is not moved, the
    others take the free places, the recent ones follow in their order; keys,
    values and weights move alike. Sequences must not share the pages of their
    first `budget` tokens."""
    who = "cache_evict"
    shape = (cache.layers, seqs.seqs, cache.heads)
    _need(keep.dim() == 4 and keep.shape[:3] == shape and keep.dtype == _ints()[0] and keep.is_contiguous(), who,
          "keep must be contiguous int32 %s + [budget]" % (shape,))
    _of_weights(weights, cache, seqs, who)
    _check(_lib().kr_op_cache_evict(cache, seqs, weights, keep.shape[3], sinks, recent, keep.data_ptr(),
                                    _launch_stream(stream, who, cache.device, seqs.device, keep)))


def _vocab_rows(t, who, name):
    """Row stride of a [rows, vocab] tensor with contiguous rows."""
    _need(t.dim() == 2 and t.shape[1] > 0 and (t.shape[1] == 1 or t.stride(1) == 1), who,
          "%s must be [rows, vocab] with contiguous rows" % name)
    return _pitch(t, who, name)


def _drafts(seqs, logits, draft, who):
    ld = _vocab_rows(logits, who, "logits")
    _need(logits.shape[0] < 1 << 31 and logits.shape[1] < 1 << 31, who, "logits are too large")
    ld_draft = 0
    if draft is not None:
        _need(draft.shape == logits.shape, who, "draft must have the logits' shape")
        ld_draft = _vocab_rows(draft, who, "draft")
    return KrDrafts(None, ld, None, ld_draft, None, None, None, None, None, _dt(logits),
                    0 if draft is None else _dt(draft), logits.shape[1], logits.shape[0])


def verify_drafts_workspace(seqs, logits, draft=None):
    """(workspace bytes, counters) that verify_drafts needs for these shapes."""
    b, c = ctypes.c_size_t(0), ctypes.c_int(0)
    _check(_lib().kr_op_verify_drafts_workspace(_drafts(seqs, logits, draft, "verify_drafts_workspace"), seqs,
                                                ctypes.byref(b), ctypes.byref(c)))
    return b.value, c.value


def verify_drafts(seqs, logits, tokens, u, u_next, path, path_lens, next_tokens, ws, counters, parents=None, draft=None,
                  temperature=None, stream=None):
    """Holds drafted tokens against the target's logits [rows, vocab] (bf16,
    f16 or f32; row r's are for the token after row r) by rejection sampling.
    The first row of each sequence is its last token, the others are drafts:
    tokens [rows] int64, each following row parents[row] of its sequence (int32
    [rows], an earlier one; None: the row before). draft [rows, vocab]: the
    probabilities from which the drafts after row r were drawn; None: they were
    not drawn. u [rows] and u_next [seqs] float32: uniform numbers in [0, 1).
    temperature [seqs] float32 (None: 1; 0: the first of the largest logits).
    Out: path [seqs, width] int32 (accepted rows from 0 on, then -1: what
    cache_compact takes; `width` rows at most), path_lens [seqs] int32,
    next_tokens [seqs] int64 (the token after the last accepted row; -1: none).
    ws (uint8) and counters (int32, zero before the first call): of
    verify_drafts_workspace's sizes, for one stream at a time."""
    who = "verify_drafts"
    d = _drafts(seqs, logits, draft, who)
    rows, n, (i32, i64), f32 = d.rows, seqs.seqs, _ints(), _f32()
    d.logits, d.draft = logits.data_ptr(), None if draft is None else draft.data_ptr()
    d.tokens, d.u = _vector(tokens, i64, rows, who, "tokens"), _vector(u, f32, rows, who, "u")
    d.u_next = _vector(u_next, f32, n, who, "u_next")
    if parents is not None:
        # (an empty tensor's address is 0, which would say that there is none)
        d.parents = _vector(parents, i32, rows, who, "parents") or 16
    if temperature is not None:
        d.temperature = _vector(temperature, f32, n, who, "temperature")
    _need(path.dim() == 2 and path.dtype == i32 and path.shape[0] == n and path.shape[1] > 0
          and (path.shape[1] == 1 or path.stride(1) == 1), who, "path must be int32 [seqs, width] with contiguous rows")
    _need(counters.dtype == i32 and counters.dim() == 1 and counters.is_contiguous() and ws.is_contiguous(), who,
          "ws and counters (an int32 vector) must be contiguous")
    _check(_lib().kr_op_verify_drafts(d, seqs, path.data_ptr(), _pitch(path, who, "path"), path.shape[1],
                                      _vector(path_lens, i32, n, who, "path_lens"),
                                      _vector(next_tokens, i64, n, who, "next_tokens"), ws.data_ptr(), ws.nbytes,
                                      counters.data_ptr(), counters.shape[0],
                                      _launch_stream(stream, who, seqs.device, seqs.device, logits, draft, tokens,
                                                     parents, u, u_next, temperature, path, path_lens, next_tokens, ws,
                                                     counters)))
