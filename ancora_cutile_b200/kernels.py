"""Thin Python wrappers over the kernel-level C entry points (one call = one or a
few kernel launches on the given stream, no synchronisation).  Arguments are device
buffers (anything ``dev_ptr`` accepts)."""
import ctypes as C

import numpy as np

from . import _lib as L
from .buffers import dev_ptr, get_context, view_span

_GRAD = {"bf16": L.GRAD_BF16, "f32": L.GRAD_F32}


def _coeff_array(coeffs):
    flat = [float(x) for t in coeffs for x in t]
    return (C.c_float * max(len(flat), 1))(*flat)


def ns_gemm_phase(mode, P, Q, Cout, E, M, N, alpha=0.0, beta=1.0, stream=None, ctx=None):
    """mode 0: C=RNE(P P^T); 1: C=RNE(alpha P + beta P P^T); 2: C=RNE(alpha Q + beta P Q)."""
    ctx = ctx or get_context()
    L.check(L.lib().anc_ns_gemm_phase(ctx.handle, int(mode), dev_ptr(P), dev_ptr(Q), dev_ptr(Cout),
                                      int(E), int(M), int(N), float(alpha), float(beta),
                                      C.c_void_p(stream or None)))


def muon_momentum(buf, g, u, K, N, momentum, nesterov=True, transposed=False, grad_dtype="bf16",
                  stream=None, ctx=None):
    ctx = ctx or get_context()
    L.check(L.lib().anc_muon_momentum(ctx.handle, dev_ptr(buf), dev_ptr(g), _GRAD[grad_dtype], dev_ptr(u),
                                      int(K), int(N), float(momentum), int(bool(nesterov)),
                                      int(bool(transposed)), C.c_void_p(stream or None)))


def muon_update(p32, p16, O, K, N, lr_scale, transposed=False, stream=None, ctx=None):
    ctx = ctx or get_context()
    L.check(L.lib().anc_muon_update(ctx.handle, dev_ptr(p32), dev_ptr(p16), dev_ptr(O), int(K), int(N),
                                    float(np.float32(lr_scale)), int(bool(transposed)),
                                    C.c_void_p(stream or None)))


def fro_normalize(X, recip, E, M, N, eps=1e-7, stream=None, ctx=None):
    ctx = ctx or get_context()
    L.check(L.lib().anc_fro_normalize(ctx.handle, dev_ptr(X), dev_ptr(recip), int(E), int(M), int(N),
                                      float(eps), C.c_void_p(stream or None)))


def ns_batched(X, A, B, Y, recip, E, M, N, steps, coeffs, eps=1e-7, stream=None, ctx=None, single_launch=True):
    """single_launch=False forces one launch per phase (same bits)."""
    ctx = ctx or get_context()
    L.check(L.lib().anc_ns_batched_ex(ctx.handle, dev_ptr(X), dev_ptr(A), dev_ptr(B), dev_ptr(Y),
                                      dev_ptr(recip), int(E), int(M), int(N), int(steps),
                                      _coeff_array(coeffs), float(eps), int(bool(single_launch)),
                                      C.c_void_p(stream or None)))


def grad_accumulate(acc, src=None, g16=None, numel=None, src_dtype="f32", elem_offset=0, scale=1.0,
                    rounding="rne", seed=0, step=0, zero_after=False, stream=None, ctx=None):
    """acc = src + acc (float32; src f32 or bf16, optional) and, in the same sweep,
    g16 = bf16(acc * scale) (optional; "rne" or "sr"), then acc = 0 when ``zero_after``.
    The accumulate sweep and the downcast the reference runs separately
    (ancora/kernels/fused.py:242-249, 144-161)."""
    ctx = ctx or get_context()
    if numel is None:
        numel = int(np.prod(acc.shape))
    L.check(L.lib().anc_grad_accumulate(ctx.handle, dev_ptr(acc), dev_ptr(src), _GRAD[src_dtype], dev_ptr(g16),
                                        int(numel), int(elem_offset), float(np.float32(scale)),
                                        {"rne": L.ROUND_RNE, "sr": L.ROUND_SR}[rounding], int(seed), int(step),
                                        int(bool(zero_after)), C.c_void_p(stream or None)))


_IDS = {"i32": L.IDS_I32, "i64": L.IDS_I64}
_SIZE = {"bf16": 2, "f32": 4, "i32": 4, "i64": 8}


def _buf(obj, rows, ld, D, dtype, what):
    """Address of ``obj``; a buffer that knows its size must hold the rows it is said to, a strided view span them."""
    if type(obj) is int:
        return obj
    n = getattr(obj, "nbytes", None)
    if n is not None and rows > 0:
        need = ((rows - 1) * (ld or D) + D) * _SIZE[dtype]
        if n < need:
            span = view_span(obj)
            n = n if span is None else span
        if n < need:
            raise ValueError(f"{what} holds {n} bytes: too few for {rows} rows of {D} {dtype}, {ld or D} elements apart")
    return dev_ptr(obj)


_EMBED = {"write": L.EMBED_WRITE, "add": L.EMBED_ADD}
_VOUCHED = 2 ** 64 - 1


def embedding_lookup(table, ids, out, T, V, D, scale=1.0, table_dtype="bf16", out_dtype="bf16", ids_dtype="i64",
                     table_ld=0, out_ld=0, stream=None, ctx=None):
    """out[t] = round(scale * table[ids[t]]) for T tokens over a (V, D) table; rows ``*_ld`` elements apart
    (0: D).  A negative id gives a zero row; an id >= V too, and sets status bit 0x8."""
    ctx = ctx or get_context()
    rc = L.lib().anc_embedding_lookup(ctx.handle, _buf(table, V, table_ld, D, table_dtype, "table"),
                                      _GRAD[table_dtype], table_ld, _buf(ids, 1, T, T, ids_dtype, "ids"),
                                      _IDS[ids_dtype], _buf(out, T, out_ld, D, out_dtype, "out"), _GRAD[out_dtype],
                                      out_ld, T, V, D, scale, stream or None)
    if rc:
        L.check(rc)


def embedding_grad_workspace(T, V, D):
    """Bytes of scratch ``embedding_grad`` needs for T tokens over a (V, D) table."""
    n = C.c_uint64()
    L.check(L.lib().anc_embedding_grad_workspace(int(T), int(V), int(D), C.byref(n)))
    return n.value


def embedding_grad(dy, ids, dw, T, V, D, work, scale=1.0, dy_dtype="bf16", dw_dtype="bf16", ids_dtype="i64",
                   mode="write", padding_idx=None, dy_ld=0, dw_ld=0, work_bytes=None, stream=None, ctx=None):
    """The embedding's gradient: dw[v] = round(scale * S_v) over the whole (V, D) table (mode "write") or
    dw[v] = round(dw[v] + scale * S_v) on the rows some token names (mode "add"), with S_v the float32 sum of
    dy[t] over the tokens with ids[t] == v, in an order the ids alone fix.  Negative ids and ``padding_idx``
    contribute nothing.  ``work``: a device buffer of ``embedding_grad_workspace(T, V, D)`` bytes that no
    other call in flight uses; ``work_bytes`` defaults to its ``nbytes``; a bare address is taken to be enough."""
    ctx = ctx or get_context()
    if work_bytes is None:
        work_bytes = getattr(work, "nbytes", _VOUCHED)
    rc = L.lib().anc_embedding_grad(ctx.handle, _buf(dy, T, dy_ld, D, dy_dtype, "dy"), _GRAD[dy_dtype], dy_ld,
                                    _buf(ids, 1, T, T, ids_dtype, "ids"), _IDS[ids_dtype],
                                    _buf(dw, V, dw_ld, D, dw_dtype, "dw"), _GRAD[dw_dtype], dw_ld, T, V, D, scale,
                                    _EMBED[mode],
                                    -1 if padding_idx is None else padding_idx, dev_ptr(work), work_bytes,
                                    stream or None)
    if rc:
        L.check(rc)
