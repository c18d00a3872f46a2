"""Floating-point operators over packed rows, with their gradients (include/nxg_rows.h): rotary
positions, layer norm and attention, in 16-bit types (rope and norm in fp32 too).

Rows of several heads are tensors [T][n_head][head_dim] with any strides whose last is 1 (a slice of a
fused projection, or head-major storage as a transposed view). Documents are given by cu_offsets, a host
sequence or a device int32 tensor, with empty documents allowed. Every function takes the streams and
raises the errors that the package's other functions do, and keeps nothing between calls.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional

import numpy as np

from . import (TYPE_BF16, TYPE_F16, TYPE_F32, _check, _device_offsets, _np_ptr, _order_on, _raw_device, _stream_ptr, _torch,
               load_library)

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


# The checks below are most of what a call for a few rows costs (10 to 20 us in all), so they look at each
# tensor once, and struct nxg_rows are made several at a time, as an array of their 64-bit words.
_types = {}
_words = {n: ctypes.c_int64 * (3 * n) for n in (2, 4, 8)}
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
    dev = t.get_device() if t.is_cuda else -1
    if dev < 0 or dev != _raw_device():
        raise ValueError(f"{name} must be a tensor on the current device")
    return dev


def _head_rows(t, name, dev, dtype, shape=None):
    """A [T][n_head][head_dim] tensor as the words of struct nxg_rows."""
    if not t.is_cuda or t.get_device() != dev:
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
    if not t.is_cuda or t.get_device() != dev:
        raise ValueError(f"{name} must be a tensor on the current device")
    if t.dtype not in dtypes or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor [{n}] of {' or '.join(map(str, dtypes))}")
    return t.data_ptr()


def _plain_rows(t, name, dev, like=None):
    """A [T][C] tensor with values next to each other: (pointer, row stride)."""
    if not t.is_cuda or t.get_device() != dev:
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
