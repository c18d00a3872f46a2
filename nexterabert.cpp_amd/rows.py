"""Floating-point operators over packed rows, with their gradients (include/nxg_rows.h): rotary
positions, layer norm, attention, head norms with rotation, dropout and low-rank adapters, in 16-bit types (all but
attention in fp32 too).

Rows of several heads are tensors [T][n_head][head_dim] with any strides whose last is 1 (a slice of a
fused projection, or head-major storage as a transposed view). Documents are given by cu_offsets, a host
sequence or a device int32 tensor, with empty documents allowed. Rows of no document are not written by attention_rows, adapter_rows
and their gradients: an output that the call makes holds anything there. Every function takes the streams and
raises the errors that the package's other functions do, and keeps nothing between calls.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional

import numpy as np

from . import (TYPE_BF16, TYPE_F16, TYPE_F32, _check, _device_offsets, _np_ptr, _order_on, _raw_device, _stream_ptr, _torch,
               _uploaded, load_library)

ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "by_parts": 3}
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}


class _Rows(ctypes.Structure):
    """struct nxg_rows."""
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _AttentionParams(ctypes.Structure):
    """struct nxg_attention_rows_params."""
    _fields_ = [("type", ctypes.c_int32), ("n_head", ctypes.c_int32), ("n_kv_head", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("T_q", ctypes.c_int32), ("T_k", ctypes.c_int32), ("n_seqs", ctypes.c_int32),
                ("cu_q", ctypes.c_void_p), ("cu_k", ctypes.c_void_p), ("left", ctypes.c_int32), ("right", ctypes.c_int32),
                ("scale", ctypes.c_float)]


# struct nxg_qk_norm_rope_params: type, T, n_head, n_kv_head, head_dim, wq, wk, w_type, eps, freq, n_rot, layout, mscale, positions,
# cu, n_seqs; struct nxg_adapter_rows_params: type, w_type, T, n_in, n_out, rank, n_adapters, n_seqs, cu, ids, a, b, scale
_qk_params = struct.Struct("@5i2PifPiif2Pi0q")
_adapter_params = struct.Struct("@8i4Pf0q")
_row = struct.Struct("@P2q")       # struct nxg_rows


# The checks below are most of what a call for a few rows costs (10 to 20 us in all), so they look at each
# tensor once, and struct nxg_rows are made several at a time, as an array of their 64-bit words.
_types = {}
_words = {n: ctypes.c_int64 * (3 * n) for n in (2, 4, 6, 8)}
_ROWS_BYTES = ctypes.sizeof(_Rows)


_INT32 = (1 << 31) - 1


def _sizes(*sizes):
    """Refuses sizes that the C functions' int32 would take modulo 2^32."""
    if max(sizes) > _INT32:
        raise ValueError(f"sizes {', '.join(map(str, sizes))}: too large")


def _side(n):
    """A window's side as an int32: past it there is no more to see."""
    n = int(n)
    return n if -_INT32 <= n <= _INT32 else _INT32 if n > 0 else -_INT32


def _type_of(t, name, allowed=None):
    if not _types:
        torch = _torch()
        _types.update({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16})
    ty = _types.get(t.dtype)
    if ty is None or (allowed is not None and ty not in allowed):
        raise ValueError(f"{name} has type {t.dtype}, which this function does not take")
    return ty


def _device_of(t, name) -> int:
    """The tensor's device, which must be the current one."""
    dev = t.get_device()           # -1: host memory
    if dev < 0 or dev != _raw_device():
        raise ValueError(f"{name} must be a tensor on the current device")
    return dev


def _head_rows(t, name, dev, dtype, shape=None):
    """A [T][n_head][head_dim] tensor as the words of struct nxg_rows."""
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a tensor on the current device")
    st = t.stride()
    if len(st) != 3 or (st[2] != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [T][n_head][head_dim] with values next to each other")
    if t.dtype != dtype:
        raise ValueError(f"{name} must have type {dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr(), st[0], st[1]


def _vector(t, name, n, dev, dtypes):
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a tensor on the current device")
    if t.dtype not in dtypes or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor [{n}] of {' or '.join(map(str, dtypes))}")
    return t.data_ptr()


def _float(x, name) -> float:
    """A number that a 32-bit float can be."""
    x = float(x)
    if not -3.4e38 <= x <= 3.4e38:
        raise ValueError(f"{name} must be a finite number that a 32-bit float holds")
    return x


def _plain_rows(t, name, dev, like=None):
    """A [T][C] tensor with values next to each other: (pointer, row stride)."""
    if t.get_device() != dev:
        raise ValueError(f"{name} must be a tensor on the current device")
    st = t.stride()
    if len(st) != 2 or (st[1] != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be [T][C] with values next to each other")
    if like is not None and (t.dtype != like.dtype or t.shape != like.shape):
        raise ValueError(f"{name} must have type {like.dtype} and shape {tuple(like.shape)}")
    return t.data_ptr(), st[0]


def _offsets_arg(cu, like, dev):
    """cu_offsets (host sequence or device int32 tensor) as a device int32 tensor."""
    torch = _torch()
    if isinstance(cu, torch.Tensor) and cu.is_cuda and cu.get_device() == dev and cu.dtype == torch.int32 and cu.dim() == 1 \
            and cu.is_contiguous() and cu.numel() > 1:
        return cu
    return _device_offsets(cu, like.device)


# --- rotary positions --------------------------------------------------------------------------

def rope_frequencies(n_rot: int, base: float, scaling: str = "none", factor: float = 1.0, train_len: int = 0):
    """Radians per position of each of the n_rot / 2 pairs (float64 numpy array) and the factor on
    the rotated values. scaling: "none", "linear", "ntk" (the encoder's own past its trained length) or
    "by_parts" (each frequency by its turns over train_len positions)."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling must be one of {', '.join(ROPE_SCALINGS)}")
    _sizes(n_rot, train_len)
    freq = np.empty(max(n_rot, 0) // 2, np.float64)
    mscale = ctypes.c_float()
    _check(load_library().nxg_rope_frequencies(n_rot, float(base), ROPE_SCALINGS[scaling], float(factor), int(train_len),
                                               _np_ptr(freq), ctypes.byref(mscale)), "rope_frequencies")
    return freq, mscale.value


def rope_rows(x, freq, cu_offsets=None, positions=None, layout: str = "half", mscale: float = 1.0, inverse: bool = False,
              out=None, stream=None):
    """Rotary positions of x [T][n_head][head_dim] (fp32, fp16 or bf16): the first 2 * len(freq) values of
    each head in pairs (i, i + n/2) ("half") or (2i, 2i + 1) ("interleaved") turned by position *
    freq[i] and scaled by mscale; the rest copied. freq: device float64 [n / 2]. The position is the row's place
    in its document, or positions (device int32 [T]). inverse turns back: the gradient of the same
    call. out may be x."""
    torch = _torch()
    ty = _type_of(x, "x")
    dev = _device_of(x, "x")
    xr = _head_rows(x, "x", dev, x.dtype)
    T, H, D = x.shape
    half = freq.numel()
    _sizes(T, H, D, half)
    fp = _vector(freq, "freq", half, dev, (torch.float64,))
    if layout not in ROPE_LAYOUTS:
        raise ValueError(f"layout must be one of {', '.join(ROPE_LAYOUTS)}")
    if (cu_offsets is None) == (positions is None):
        raise ValueError("give either cu_offsets or positions")
    cu = None
    if positions is not None:
        pp, cp, n_seqs = _vector(positions, "positions", T, dev, (torch.int32,)), None, 0
    else:
        cu = _offsets_arg(cu_offsets, x, dev)
        pp, cp, n_seqs = None, cu.data_ptr(), cu.numel() - 1
    if out is None:
        out = x.new_empty((T, H, D))
    rows = _words[2](*xr, *_head_rows(out, "out", dev, x.dtype, x.shape))
    at = ctypes.addressof(rows)
    _order_on(stream, cu, out)
    _check(load_library().nxg_rope_rows(ty, at, T, H, D, fp, 2 * half, ROPE_LAYOUTS[layout], float(mscale), 1 if inverse else 0,
                                        pp, cp, n_seqs, at + _ROWS_BYTES, _stream_ptr(stream)), "rope_rows")
    return out


# --- layer norm --------------------------------------------------------------------------------

def _norm_weights(x, w, b, dev):
    """(w pointer, b pointer, weight type)."""
    first = w if w is not None else b
    if first is None:
        return None, None, TYPE_F32
    wt = _type_of(first, "w")
    if wt != TYPE_F32 and first.dtype != x.dtype:
        raise ValueError(f"w and b must be float32 or {x.dtype}")
    n, dtypes = x.shape[1], (first.dtype,)
    return (None if w is None else _vector(w, "w", n, dev, dtypes)), (None if b is None else _vector(b, "b", n, dev, dtypes)), wt


def layer_norm_rows(x, w=None, b=None, eps: float = 1e-5, out=None, mean=None, rstd=None, stream=None):
    """Layer norm of the rows of x [T][C] (fp32, fp16 or bf16), times w plus b (of x's type or fp32; either
    may be None). Returns (y, mean, rstd), the last two fp32 [T], as layer_norm_rows_backward takes them. out
    may be x."""
    torch = _torch()
    ty = _type_of(x, "x")
    dev = _device_of(x, "x")
    xp, xs = _plain_rows(x, "x", dev)
    T, C = x.shape
    _sizes(T, C)
    wp, bp, wt = _norm_weights(x, w, b, dev)
    if out is None:
        out = x.new_empty((T, C))
    yp, ys = _plain_rows(out, "out", dev, x)
    f32 = torch.float32
    if mean is None and rstd is None:
        mean, rstd = x.new_empty((2, T), dtype=f32)
    else:
        mean = x.new_empty(T, dtype=f32) if mean is None else mean
        rstd = x.new_empty(T, dtype=f32) if rstd is None else rstd
    mp, rp = _vector(mean, "mean", T, dev, (f32,)), _vector(rstd, "rstd", T, dev, (f32,))
    _order_on(stream, out, mean, rstd)
    _check(load_library().nxg_layer_norm_rows(ty, xp, xs, wp, bp, wt, float(eps), T, C, yp, ys, mp, rp, _stream_ptr(stream)),
           "layer_norm_rows")
    return out, mean, rstd


@functools.lru_cache(maxsize=256)
def layer_norm_rows_workspace_bytes(T: int, C: int) -> int:
    """nxg_layer_norm_rows_workspace_bytes."""
    _sizes(T, C)
    n = int(load_library().nxg_layer_norm_rows_workspace_bytes(T, C))
    _check(-n if n < 0 else 0, "layer_norm_rows_workspace_bytes")
    return n


def _workspace(t, nbytes, like):
    """The caller's workspace (a uint8 device tensor) or one made for the call."""
    torch = _torch()
    if t is None:
        return like.new_empty(nbytes, dtype=torch.uint8)
    if not t.is_cuda or t.get_device() != like.get_device():
        raise ValueError("workspace must be a tensor on the current device")
    if t.dtype != torch.uint8 or not t.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 device tensor")
    return t


def layer_norm_rows_backward(dy, x, mean, rstd, w=None, dx=None, dw=None, db=None, workspace=None, stream=None):
    """The gradients of layer_norm_rows: (dx, dw, db), dw and db of w's type (fp32 without w).
    workspace: None (made for the call) or a uint8 device tensor of layer_norm_rows_workspace_bytes(T, C)."""
    torch = _torch()
    ty = _type_of(x, "x")
    dev = _device_of(x, "x")
    xp, xs = _plain_rows(x, "x", dev)
    gp, gs = _plain_rows(dy, "dy", dev, x)
    T, C = x.shape
    _sizes(T, C)
    wp, _, wt = _norm_weights(x, w, None, dev)
    f32 = (torch.float32,)
    w_dtype = w.dtype if w is not None else f32[0]
    mp, rp = _vector(mean, "mean", T, dev, f32), _vector(rstd, "rstd", T, dev, f32)
    if dx is None:
        dx = x.new_empty((T, C))
    dxp, dxs = _plain_rows(dx, "dx", dev, x)
    dw = x.new_empty(C, dtype=w_dtype) if dw is None else dw
    db = x.new_empty(C, dtype=w_dtype) if db is None else db
    dwp, dbp = _vector(dw, "dw", C, dev, (w_dtype,)), _vector(db, "db", C, dev, (w_dtype,))
    ws = _workspace(workspace, layer_norm_rows_workspace_bytes(T, C), x)
    _order_on(stream, dx, dw, db, ws)
    _check(load_library().nxg_layer_norm_rows_backward(ty, gp, gs, xp, xs, mp, rp, wp, wt, T, C, dxp, dxs, dwp, dbp,
                                                       ws.data_ptr(), ws.numel(), _stream_ptr(stream)), "layer_norm_rows_backward")
    return dx, dw, db


# --- attention ---------------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _attention_bytes(dev, ty, H, G, D, T, K, n_seqs, left, right):
    """The workspaces of the two passes for these sizes on this device (the scale has no part in them)."""
    L = load_library()
    p = ctypes.byref(_AttentionParams(ty, H, G, D, T, K, n_seqs, None, None, left, right, 1.0))
    n = int(L.nxg_attention_rows_workspace_bytes(p)), int(L.nxg_attention_rows_backward_workspace_bytes(p))
    _check(-min(n) if min(n) < 0 else 0, "attention_rows")
    return n


def _attention_args(q, k, v, cu_q, cu_k, left, right, scale):
    """(params, the words of q, k and v, workspaces, cu_q, cu_k, device)"""
    ty = _type_of(q, "q", (TYPE_F16, TYPE_BF16))
    dev, dtype = _device_of(q, "q"), q.dtype
    words = _head_rows(q, "q", dev, dtype) + _head_rows(k, "k", dev, dtype) + _head_rows(v, "v", dev, dtype, k.shape)
    T, H, D = q.shape
    K, G, Dk = k.shape
    if Dk != D:
        raise ValueError(f"k and v must have heads of {D}")
    _sizes(T, H, K, G, D)
    cu_q = _offsets_arg(cu_q, q, dev)
    cu_k = cu_q if cu_k is None else _offsets_arg(cu_k, q, dev)
    n = cu_q.numel()
    if cu_k.numel() != n:
        raise ValueError("cu_q and cu_k must have the same number of documents")
    left, right = _side(left), _side(right)
    sizes = _attention_bytes(dev, ty, H, G, D, T, K, n - 1, left, right)
    p = _AttentionParams(ty, H, G, D, T, K, n - 1, cu_q.data_ptr(), cu_k.data_ptr(), left, right,
                         1.0 / math.sqrt(D) if scale is None else float(scale))
    return p, words, sizes, cu_q, cu_k, dev


def _lse_arg(lse, T, H, dev):
    if not lse.is_cuda or lse.get_device() != dev:
        raise ValueError("lse must be a tensor on the current device")
    if lse.dtype != _torch().float32 or lse.shape != (T, H) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 tensor [{T}][{H}]")
    return lse.data_ptr()


def attention_rows(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1, right: int = -1, out=None, lse=None,
                   workspace=None, stream=None):
    """Grouped-query attention inside each document: q [T_q][n_head][head_dim], k and v
    [T_k][n_kv_head][head_dim] (fp16 or bf16, head_dim a multiple of 8 up to 128), cu_k None for the
    queries' own documents. Query i of n stands at key i + m - n of m and sees the keys from left before to
    right behind it (-1: no limit; right=0: causal; left=right=h: a sliding window). Returns (out, lse), lse the
    fp32 [T_q][n_head] log of each query's sum, as attention_rows_backward takes it. Queries without a key
    give 0 and -inf. workspace: None (made where the launch uses one) or a uint8 device tensor."""
    torch = _torch()
    p, words, sizes, cu_q, cu_k, dev = _attention_args(q, k, v, cu_q, cu_k, left, right, scale)
    T, H, _ = q.shape
    if out is None:
        out = q.new_empty(q.shape)
    if lse is None:
        lse = q.new_empty((T, H), dtype=torch.float32)
    lp = _lse_arg(lse, T, H, dev)
    rows = _words[4](*words, *_head_rows(out, "out", dev, q.dtype, q.shape))
    at = ctypes.addressof(rows)
    ws = _workspace(workspace, sizes[0], q) if sizes[0] or workspace is not None else None
    n = 0 if ws is None else ws.numel()
    _order_on(stream, cu_q, cu_k, out, lse, ws)
    _check(load_library().nxg_attention_rows(ctypes.byref(p), at, at + _ROWS_BYTES, at + 2 * _ROWS_BYTES, at + 3 * _ROWS_BYTES, lp,
                                             ws.data_ptr() if n else None, n, _stream_ptr(stream)), "attention_rows")
    return out, lse


def attention_rows_backward_workspace_bytes(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1, right: int = -1) -> int:
    """The workspace attention_rows_backward takes for these arguments."""
    return _attention_args(q, k, v, cu_q, cu_k, left, right, scale)[2][1]


def attention_rows_backward(dout, q, k, v, out, lse, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1,
                            right: int = -1, dq=None, dk=None, dv=None, workspace=None, stream=None):
    """The gradients of attention_rows: (dq, dk, dv), from dout, its inputs and what it returned (out, lse).
    Rows of no document are left as they were. workspace: None (made for the call) or a uint8 device tensor of
    attention_rows_backward_workspace_bytes."""
    p, words, sizes, cu_q, cu_k, dev = _attention_args(q, k, v, cu_q, cu_k, left, right, scale)
    T, H, _ = q.shape
    dtype = q.dtype
    lp = _lse_arg(lse, T, H, dev)
    dq = q.new_empty(q.shape) if dq is None else dq
    dk = q.new_empty(k.shape) if dk is None else dk
    dv = q.new_empty(k.shape) if dv is None else dv
    rows = _words[8](*words, *_head_rows(dout, "dout", dev, dtype, q.shape), *_head_rows(out, "out", dev, dtype, q.shape),
                     *_head_rows(dq, "dq", dev, dtype, q.shape), *_head_rows(dk, "dk", dev, dtype, k.shape),
                     *_head_rows(dv, "dv", dev, dtype, k.shape))
    qa, ka, va, da, oa, dqa, dka, dva = range(ctypes.addressof(rows), ctypes.addressof(rows) + 8 * _ROWS_BYTES, _ROWS_BYTES)
    ws = _workspace(workspace, sizes[1], q)
    _order_on(stream, cu_q, cu_k, dq, dk, dv, ws)
    _check(load_library().nxg_attention_rows_backward(ctypes.byref(p), da, qa, ka, va, oa, lp, dqa, dka, dva, ws.data_ptr(),
                                                      ws.numel(), _stream_ptr(stream)), "attention_rows_backward")
    return dq, dk, dv


# --- norms of queries and keys, and their rotation -----------------------------------------------

def _qk_args(q, k, wq, wk, freq, cu_offsets, positions, eps, layout, mscale):
    """(params, q's and k's struct nxg_rows, cu, device)"""
    torch = _torch()
    dtype = q.dtype
    ty, dev = _type_of(q, "q"), _device_of(q, "q")
    qr = _row.pack(*_head_rows(q, "q", dev, dtype))
    T, H, D = q.shape
    half = freq.numel()
    if (k is None) != (wk is None):
        raise ValueError("give k and wk together")
    G, kr = 0, None
    if k is not None:
        kr = _row.pack(*_head_rows(k, "k", dev, dtype))
        Tk, G, Dk = k.shape
        if Tk != T or Dk != D or G == 0:
            raise ValueError(f"k must have shape ({T}, n_kv_head, {D})")
    _sizes(T, H, G, D, half)
    wdtype = wq.dtype
    wt = _type_of(wq, "wq")
    if wt != TYPE_F32 and wdtype != dtype:
        raise ValueError(f"wq and wk must be float32 or {dtype}")
    qw = _vector(wq, "wq", D, dev, (wdtype,))
    kw = 0 if k is None else _vector(wk, "wk", D, dev, (wdtype,))
    fp = _vector(freq, "freq", half, dev, (torch.float64,))
    if layout not in ROPE_LAYOUTS:
        raise ValueError(f"layout must be one of {', '.join(ROPE_LAYOUTS)}")
    if (cu_offsets is None) == (positions is None):
        raise ValueError("give either cu_offsets or positions")
    cu, pp, cp, n_seqs = None, 0, 0, 0
    if positions is not None:
        pp = _vector(positions, "positions", T, dev, (torch.int32,))
    else:
        cu = _offsets_arg(cu_offsets, q, dev)
        cp, n_seqs = cu.data_ptr(), cu.numel() - 1
    p = _qk_params.pack(ty, T, H, G, D, qw, kw, wt, _float(eps, "eps"), fp, 2 * half, ROPE_LAYOUTS[layout], _float(mscale, "mscale"),
                        pp, cp, n_seqs)
    return p, qr, kr, cu, dev


def _rows_out(t, name, dev, like):
    """(t, its struct nxg_rows): rows of the shape and type of `like`, made where t is None."""
    if t is None:
        t = like.new_empty(like.shape)
        return t, _row.pack(t.data_ptr(), *t.stride()[:2])
    return t, _row.pack(*_head_rows(t, name, dev, like.dtype, like.shape))


def qk_norm_rope_rows(q, k, wq, wk, freq, cu_offsets=None, positions=None, eps: float = 1e-6, layout: str = "half",
                      mscale: float = 1.0, q_out=None, k_out=None, stream=None):
    """The RMS norm of every head of q [T][n_head][head_dim] and k [T][n_kv_head][head_dim] (fp32, fp16 or bf16), times wq or
    wk [head_dim] (of their type or fp32), then rotary positions as rope_rows turns them: for layers whose heads have RMS norms
    (the encoder's own have qkv_prep's tanh there). k and wk may both be None. Returns
    (q_out, k_out), which may be q and k."""
    p, qr, kr, cu, dev = _qk_args(q, k, wq, wk, freq, cu_offsets, positions, eps, layout, mscale)
    q_out, qo = _rows_out(q_out, "q_out", dev, q)
    k_out, ko = (None, None) if k is None else _rows_out(k_out, "k_out", dev, k)
    _order_on(stream, cu, q_out, k_out)
    _check(load_library().nxg_qk_norm_rope_rows(p, qr, kr, qo, ko, _stream_ptr(stream)), "qk_norm_rope_rows")
    return q_out, k_out


@functools.lru_cache(maxsize=256)
def qk_norm_rope_rows_workspace_bytes(head_dim: int) -> int:
    """The workspace qk_norm_rope_rows_backward takes for heads of this size."""
    _sizes(head_dim)
    p = _qk_params.pack(TYPE_F32, 0, 1, 0, head_dim, 0, 0, TYPE_F32, 0.0, 0, 2, 0, 1.0, 0, 0, 0)
    n = int(load_library().nxg_qk_norm_rope_rows_workspace_bytes(p))
    _check(-n if n < 0 else 0, "qk_norm_rope_rows_workspace_bytes")
    return n


def qk_norm_rope_rows_backward(dq_out, dk_out, q, k, wq, wk, freq, cu_offsets=None, positions=None, eps: float = 1e-6,
                               layout: str = "half", mscale: float = 1.0, dq=None, dk=None, dwq=None, dwk=None, workspace=None,
                               stream=None):
    """The gradients of qk_norm_rope_rows: (dq, dk, dwq, dwk), from the gradients of its outputs and its inputs; dwq and dwk of
    wq's type. dq may be dq_out or q, dk dk_out or k. Without k and wk: dk and dwk are None. workspace: None (made for the
    call) or a uint8 device tensor of qk_norm_rope_rows_workspace_bytes(head_dim)."""
    p, qr, kr, cu, dev = _qk_args(q, k, wq, wk, freq, cu_offsets, positions, eps, layout, mscale)
    D = q.shape[2]
    gq = _row.pack(*_head_rows(dq_out, "dq_out", dev, q.dtype, q.shape))
    dq, dqr = _rows_out(dq, "dq", dev, q)
    dwq = q.new_empty(D, dtype=wq.dtype) if dwq is None else dwq
    wqp, wkp, gk, dkr = _vector(dwq, "dwq", D, dev, (wq.dtype,)), None, None, None
    if k is None:
        dk = dwk = None
    else:
        gk = _row.pack(*_head_rows(dk_out, "dk_out", dev, q.dtype, k.shape))
        dk, dkr = _rows_out(dk, "dk", dev, k)
        dwk = q.new_empty(D, dtype=wq.dtype) if dwk is None else dwk
        wkp = _vector(dwk, "dwk", D, dev, (wq.dtype,))
    ws = _workspace(workspace, qk_norm_rope_rows_workspace_bytes(D), q)
    _order_on(stream, cu, dq, dk, dwq, dwk, ws)
    _check(load_library().nxg_qk_norm_rope_rows_backward(p, gq, gk, qr, kr, dqr, dkr, wqp, wkp, ws.data_ptr(), ws.numel(),
                                                         _stream_ptr(stream)), "qk_norm_rope_rows_backward")
    return dq, dk, dwq, dwk


# --- dropout -------------------------------------------------------------------------------------

def dropout_rows(x, p: float, seed: int, offset: int = 0, step=None, residual=None, out=None, stream=None):
    """residual + dropout(x) of rows x [T][C] (fp32, fp16 or bf16); residual None: dropout alone. Which values are kept is drawn
    again by every call from (seed, offset, row, column): dropout_rows(dout, p, seed, offset) is the gradient of x. Kept values are
    divided by 1 - p (p a multiple of 2^-16, or rounded to one). seed and offset: 0 .. 2^64 - 1; step: a device int64 [1] that is added to offset when the call
    runs (new masks in the replays of a graph). out may be x or residual."""
    ty = _type_of(x, "x")
    dev = _device_of(x, "x")
    xp, xs = _plain_rows(x, "x", dev)
    T, C = x.shape
    _sizes(T, C)
    rp, rs = (None, 0) if residual is None else _plain_rows(residual, "residual", dev, x)
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("seed and offset must be 64-bit numbers")
    sp = None if step is None else _vector(step, "step", 1, dev, (_torch().int64,))
    if out is None:
        out = x.new_empty((T, C))
        op, os_ = out.data_ptr(), C
    else:
        op, os_ = _plain_rows(out, "out", dev, x)
    _order_on(stream, out)
    _check(load_library().nxg_dropout_rows(ty, xp, xs, rp, rs, T, C, float(p), seed, offset, sp, op, os_, _stream_ptr(stream)),
           "dropout_rows")
    return out


# --- low-rank adapters -----------------------------------------------------------------------------

@functools.lru_cache(maxsize=256)
def _adapter_bytes(dev, ty, wt, T, K, N, r, n, n_seqs):
    """The backward pass's workspace for these sizes on this device."""
    p = _adapter_params.pack(ty, wt, T, K, N, r, n, n_seqs, 0, 0, 0, 0, 1.0)
    b = int(load_library().nxg_adapter_rows_backward_workspace_bytes(p))
    _check(-b if b < 0 else 0, "adapter_rows_backward")
    return b


def _ids_arg(ids, n_seqs, like, dev):
    """ids (host sequence or tensor, or device int32 tensor) as a device int32 tensor [n_seqs]."""
    torch = _torch()
    if not isinstance(ids, torch.Tensor) or (ids.device.type == "cpu" and not ids.is_floating_point()):
        host = np.ascontiguousarray(ids)
        if host.ndim == 1 and host.shape[0] == n_seqs and host.dtype.kind in "iu":
            return _uploaded(np.clip(host, -1, _INT32).astype(np.int32), like.device)
    elif ids.is_cuda and ids.get_device() == dev and ids.dtype == torch.int32 and ids.dim() == 1 and ids.shape[0] == n_seqs \
            and ids.is_contiguous():
        return ids
    raise ValueError(f"ids must be {n_seqs} whole numbers: a host sequence or tensor, or a contiguous int32 tensor on the current device")


def _adapter_args(x, a, b, cu_offsets, ids, scale):
    """(params, (type, w_type, T, n_in, n_out, rank, n_adapters, n_seqs), cu, ids, device)"""
    ty, dev, wt, wdtype = _type_of(x, "x"), _device_of(x, "x"), _type_of(a, "a"), a.dtype
    if wt != ty and ty != TYPE_F32:
        raise ValueError(f"a and b must have type {x.dtype}")
    for t, name in ((a, "a"), (b, "b")):
        if t.get_device() != dev:
            raise ValueError(f"{name} must be a tensor on the current device")
        if t.dtype != wdtype or t.dim() != 3 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of 3 dimensions and type {wdtype}")
    n, r, K = a.shape
    nb, N, rb = b.shape
    if nb != n or rb != r or x.dim() != 2 or x.shape[1] != K:
        raise ValueError("x [T][n_in], a [n_adapters][rank][n_in] and b [n_adapters][n_out][rank] do not fit")
    T = x.shape[0]
    _sizes(T, K, N, r, n)
    cu = _offsets_arg(cu_offsets, x, dev)
    n_seqs = cu.numel() - 1
    ids = _ids_arg(ids, n_seqs, x, dev)
    sizes = ty, wt, T, K, N, r, n, n_seqs
    p = _adapter_params.pack(*sizes, cu.data_ptr(), ids.data_ptr(), a.data_ptr(), b.data_ptr(), _float(scale, "scale"))
    return p, sizes, cu, ids, dev


def _s_arg(s, T, r, dev):
    if not s.is_cuda or s.get_device() != dev:
        raise ValueError("s must be a tensor on the current device")
    if s.dtype != _torch().float32 or s.shape != (T, r) or not s.is_contiguous():
        raise ValueError(f"s must be a contiguous float32 tensor [{T}][{r}]")
    return s.data_ptr()


def _rows_of_width(t, name, dev, dtype, T, C):
    if t.dtype != dtype or t.shape != (T, C):
        raise ValueError(f"{name} must have type {dtype} and shape ({T}, {C})")
    return _plain_rows(t, name, dev)


def adapter_rows(x, a, b, cu_offsets, ids, scale: float = 1.0, base=None, out=None, s=None, stream=None):
    """Low-rank adapters of many requests: document d's rows of x [T][n_in] through adapter i = ids[d], base + scale * (x a_i^T)
    b_i^T, a [n_adapters][rank][n_in] and b [n_adapters][n_out][rank] of x's type (fp32 rows, as the int8 linears leave them: of any
    type). base [T][n_out]: the shared projection's rows, or None. An id that is no adapter leaves base as it is (0 without).
    Returns (out, s), s the fp32 [T][rank] rows x a_i^T, as adapter_rows_backward takes them. out may be base. Rows of no document
    are left as they were (uninitialised where the call makes out or s). ids: a host sequence or tensor, or device int32."""
    p, (_, _, T, _, N, r, _, _), cu, ids, dev = _adapter_args(x, a, b, cu_offsets, ids, scale)
    xp, xs = _plain_rows(x, "x", dev)
    bp, bs = (None, 0) if base is None else _rows_of_width(base, "base", dev, x.dtype, T, N)
    if out is None:
        out = x.new_empty((T, N))
        op, os_ = out.data_ptr(), N
    else:
        op, os_ = _rows_of_width(out, "out", dev, x.dtype, T, N)
    if s is None:
        s = x.new_empty((T, r), dtype=_torch().float32)
        sp = s.data_ptr()
    else:
        sp = _s_arg(s, T, r, dev)
    _order_on(stream, cu, ids, out, s)
    _check(load_library().nxg_adapter_rows(p, xp, xs, bp, bs, op, os_, sp, _stream_ptr(stream)), "adapter_rows")
    return out, s


def adapter_rows_backward_workspace_bytes(x, a, b, cu_offsets, ids) -> int:
    """The workspace adapter_rows_backward takes for these arguments."""
    _, sizes, _, _, dev = _adapter_args(x, a, b, cu_offsets, ids, 1.0)
    return _adapter_bytes(dev, *sizes)


def adapter_rows_backward(dout, x, a, b, s, cu_offsets, ids, scale: float = 1.0, base=None, dx=None, da=None, db=None, workspace=None,
                          stream=None):
    """The gradients of adapter_rows: (dx, da, db), from dout [T][n_out], its inputs and the s that it returned. base [T][n_in]: what
    dx is added to (the shared projection's part), or None; dx may be base. da and db as a and b, zeros for adapters
    that no row has. Rows of no document are left as they were in dx. workspace: None (made for the call) or a uint8 device tensor of
    adapter_rows_backward_workspace_bytes."""
    p, sizes, cu, ids, dev = _adapter_args(x, a, b, cu_offsets, ids, scale)
    _, _, T, K, N, r, _, _ = sizes
    xp, xs = _plain_rows(x, "x", dev)
    gp, gs = _rows_of_width(dout, "dout", dev, x.dtype, T, N)
    sp = _s_arg(s, T, r, dev)
    bp, bs = (None, 0) if base is None else _rows_of_width(base, "base", dev, x.dtype, T, K)
    dx = x.new_empty((T, K)) if dx is None else dx
    dp, ds = _rows_of_width(dx, "dx", dev, x.dtype, T, K)
    da = a.new_empty(a.shape) if da is None else da
    db = b.new_empty(b.shape) if db is None else db
    for t, like, name in ((da, a, "da"), (db, b, "db")):
        if t.get_device() != dev:
            raise ValueError(f"{name} must be a tensor on the current device")
        if t.dtype != like.dtype or t.shape != like.shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of type {like.dtype} and shape {tuple(like.shape)}")
    ws = _workspace(workspace, _adapter_bytes(dev, *sizes), x)
    _order_on(stream, cu, ids, dx, da, db, ws)
    _check(load_library().nxg_adapter_rows_backward(p, gp, gs, xp, xs, sp, bp, bs, dp, ds, da.data_ptr(), db.data_ptr(),
                                                    ws.data_ptr(), ws.numel(), _stream_ptr(stream)), "adapter_rows_backward")
    return dx, da, db
