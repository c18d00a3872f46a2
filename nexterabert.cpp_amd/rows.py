"""Floating-point operators over packed rows, with their gradients (include/nxg_rows.h): rotary
positions, layer norm and attention, in 16-bit types (rope and norm in fp32 too).

Rows of several heads are tensors [T][n_head][head_dim] with any strides whose last is 1 (a slice of a
fused projection, or head-major storage as a transposed view). Documents are given by cu_offsets, a host
sequence or a device int32 tensor, with empty documents allowed. Every function takes the streams and
raises the errors that the package's other functions do, and keeps nothing between calls.
"""
from __future__ import annotations

import ctypes
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


_types = {}


def _type_of(t, name, allowed=None):
    if not _types:
        torch = _torch()
        _types.update({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16})
    ty = _types.get(t.dtype)
    if ty is None or (allowed is not None and ty not in allowed):
        raise ValueError(f"{name} has type {t.dtype}, which this function does not take")
    return ty


def _on_current_device(t, name):
    if not t.is_cuda or t.device.index != _raw_device():
        raise ValueError(f"{name} must be a tensor on the current device")
    return t


def _head_rows(t, name, like=None, shape=None):
    """A [T][n_head][head_dim] tensor as struct nxg_rows."""
    _on_current_device(t, name)
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name} must be [T][n_head][head_dim] with values next to each other")
    if like is not None and t.dtype != like.dtype:
        raise ValueError(f"{name} must have type {like.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return _Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _vector(t, name, n, dtypes):
    _on_current_device(t, name)
    if t.dtype not in dtypes or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor [{n}] of {' or '.join(map(str, dtypes))}")
    return t.data_ptr()


def _plain_rows(t, name, like=None):
    """A [T][C] tensor with values next to each other: (pointer, row stride)."""
    _on_current_device(t, name)
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be [T][C] with values next to each other")
    if like is not None and (t.dtype != like.dtype or t.shape != like.shape):
        raise ValueError(f"{name} must have type {like.dtype} and shape {tuple(like.shape)}")
    return t.data_ptr(), t.stride(0)


# --- rotary positions --------------------------------------------------------------------------

def rope_frequencies(n_rot: int, base: float, scaling: str = "none", factor: float = 1.0, train_len: int = 0):
    """Radians per position of each of the n_rot / 2 pairs (float64 numpy array) and the factor on
    the rotated values. scaling: "none", "linear", "ntk" (the encoder's own past its trained length) or
    "by_parts" (each frequency by its turns over train_len positions)."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling must be one of {', '.join(ROPE_SCALINGS)}")
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
    xr = _head_rows(x, "x")
    T, H, D = x.shape
    n = 2 * freq.numel()
    fp = _vector(freq, "freq", n // 2, (torch.float64,))
    if layout not in ROPE_LAYOUTS:
        raise ValueError(f"layout must be one of {', '.join(ROPE_LAYOUTS)}")
    if (cu_offsets is None) == (positions is None):
        raise ValueError("give either cu_offsets or positions")
    cu = None
    if positions is not None:
        pp, cp, n_seqs = _vector(positions, "positions", T, (torch.int32,)), None, 0
    else:
        cu = _device_offsets(cu_offsets, x.device)
        pp, cp, n_seqs = None, cu.data_ptr(), cu.numel() - 1
    if out is None:
        out = torch.empty((T, H, D), dtype=x.dtype, device=x.device)
    orows = _head_rows(out, "out", x, x.shape)
    _order_on(stream, cu, out)
    _check(load_library().nxg_rope_rows(ty, ctypes.byref(xr), T, H, D, fp, n, ROPE_LAYOUTS[layout], float(mscale),
                                        1 if inverse else 0, pp, cp, n_seqs, ctypes.byref(orows), _stream_ptr(stream)), "rope_rows")
    return out


# --- layer norm --------------------------------------------------------------------------------

def _norm_weights(x, w, b):
    """(w pointer, b pointer, weight type)."""
    torch = _torch()
    given = [t for t in (w, b) if t is not None]
    wt = _type_of(given[0], "w") if given else TYPE_F32
    if given and given[-1].dtype != given[0].dtype:
        raise ValueError("w and b must have one type")
    ptr = [None if t is None else _vector(t, name, x.shape[1], (torch.float32, x.dtype)) for name, t in (("w", w), ("b", b))]
    return ptr[0], ptr[1], wt


def layer_norm_rows(x, w=None, b=None, eps: float = 1e-5, out=None, mean=None, rstd=None, stream=None):
    """Layer norm of the rows of x [T][C] (fp32, fp16 or bf16), times w plus b (of x's type or fp32; either
    may be None). Returns (y, mean, rstd), the last two fp32 [T], as layer_norm_rows_backward takes them. out
    may be x."""
    torch = _torch()
    ty = _type_of(x, "x")
    xp, xs = _plain_rows(x, "x")
    T, C = x.shape
    wp, bp, wt = _norm_weights(x, w, b)
    if out is None:
        out = torch.empty((T, C), dtype=x.dtype, device=x.device)
    yp, ys = _plain_rows(out, "out", x)
    mean = torch.empty(T, dtype=torch.float32, device=x.device) if mean is None else mean
    rstd = torch.empty(T, dtype=torch.float32, device=x.device) if rstd is None else rstd
    mp, rp = (_vector(t, name, T, (torch.float32,)) for name, t in (("mean", mean), ("rstd", rstd)))
    _order_on(stream, out, mean, rstd)
    _check(load_library().nxg_layer_norm_rows(ty, xp, xs, wp, bp, wt, float(eps), T, C, yp, ys, mp, rp, _stream_ptr(stream)),
           "layer_norm_rows")
    return out, mean, rstd


def layer_norm_rows_workspace_bytes(T: int, C: int) -> int:
    """nxg_layer_norm_rows_workspace_bytes."""
    n = int(load_library().nxg_layer_norm_rows_workspace_bytes(T, C))
    _check(-n if n < 0 else 0, "layer_norm_rows_workspace_bytes")
    return n


def _workspace(t, nbytes, device):
    """The caller's workspace (a uint8 device tensor) or one made for the call."""
    torch = _torch()
    if t is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    _on_current_device(t, "workspace")
    if t.dtype != torch.uint8 or not t.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 device tensor")
    return t


def layer_norm_rows_backward(dy, x, mean, rstd, w=None, dx=None, dw=None, db=None, workspace=None, stream=None):
    """The gradients of layer_norm_rows: (dx, dw, db), dw and db of w's type (fp32 without w).
    workspace: None (made for the call) or a uint8 device tensor of layer_norm_rows_workspace_bytes(T, C)."""
    torch = _torch()
    ty = _type_of(x, "x")
    xp, xs = _plain_rows(x, "x")
    gp, gs = _plain_rows(dy, "dy", x)
    T, C = x.shape
    wp, _, wt = _norm_weights(x, w, None)
    w_dtype = w.dtype if w is not None else torch.float32
    mp, rp = (_vector(t, name, T, (torch.float32,)) for name, t in (("mean", mean), ("rstd", rstd)))
    if dx is None:
        dx = torch.empty((T, C), dtype=x.dtype, device=x.device)
    dxp, dxs = _plain_rows(dx, "dx", x)
    dw = torch.empty(C, dtype=w_dtype, device=x.device) if dw is None else dw
    db = torch.empty(C, dtype=w_dtype, device=x.device) if db is None else db
    dwp, dbp = (_vector(t, name, C, (w_dtype,)) for name, t in (("dw", dw), ("db", db)))
    ws = _workspace(workspace, layer_norm_rows_workspace_bytes(T, C), x.device)
    _order_on(stream, dx, dw, db, ws)
    _check(load_library().nxg_layer_norm_rows_backward(ty, gp, gs, xp, xs, mp, rp, wp, wt, T, C, dxp, dxs, dwp, dbp,
                                                       ws.data_ptr(), ws.numel(), _stream_ptr(stream)), "layer_norm_rows_backward")
    return dx, dw, db


# --- attention ---------------------------------------------------------------------------------

def _attention_params(q, k, v, cu_q, cu_k, left, right, scale):
    ty = _type_of(q, "q", (TYPE_F16, TYPE_BF16))
    rows = [_head_rows(q, "q"), _head_rows(k, "k", q), _head_rows(v, "v", q, k.shape)]
    T, H, D = q.shape
    if k.shape[2] != D:
        raise ValueError(f"k and v must have heads of {D}")
    cu_q = _device_offsets(cu_q, q.device)
    cu_k = cu_q if cu_k is None else _device_offsets(cu_k, q.device)
    if cu_q.numel() != cu_k.numel():
        raise ValueError("cu_q and cu_k must have the same number of documents")
    p = _AttentionParams(ty, H, k.shape[1], D, T, k.shape[0], cu_q.numel() - 1, cu_q.data_ptr(), cu_k.data_ptr(), int(left),
                         int(right), 1.0 / math.sqrt(D) if scale is None else float(scale))
    return p, rows, cu_q, cu_k


def attention_rows(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1, right: int = -1, out=None, lse=None,
                   workspace=None, stream=None):
    """Grouped-query attention inside each document: q [T_q][n_head][head_dim], k and v
    [T_k][n_kv_head][head_dim] (fp16 or bf16, head_dim a multiple of 8 up to 128), cu_k None for the
    queries' own documents. Query i of n stands at key i + m - n of m and sees the keys from left before to
    right behind it (-1: no limit; right=0: causal; left=right=h: a sliding window). Returns (out, lse), lse the
    fp32 [T_q][n_head] log of each query's sum, as attention_rows_backward takes it. Queries without a key
    give 0 and -inf. workspace: None (made where the launch uses one) or a uint8 device tensor."""
    torch = _torch()
    L = load_library()
    p, (qr, kr, vr), cu_q, cu_k = _attention_params(q, k, v, cu_q, cu_k, left, right, scale)
    T, H, D = q.shape
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    orows = _head_rows(out, "out", q, q.shape)
    if lse is None:
        lse = torch.empty((T, H), dtype=torch.float32, device=q.device)
    elif lse.dtype != torch.float32 or tuple(lse.shape) != (T, H) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 tensor [{T}][{H}]")
    _on_current_device(lse, "lse")
    n = int(L.nxg_attention_rows_workspace_bytes(ctypes.byref(p)))
    _check(-n if n < 0 else 0, "attention_rows")
    ws = _workspace(workspace, n, q.device) if n or workspace is not None else None
    _order_on(stream, cu_q, cu_k, out, lse, ws)
    _check(L.nxg_attention_rows(ctypes.byref(p), ctypes.byref(qr), ctypes.byref(kr), ctypes.byref(vr), ctypes.byref(orows),
                                lse.data_ptr(), ws.data_ptr() if ws is not None and ws.numel() else None,
                                ws.numel() if ws is not None else 0, _stream_ptr(stream)), "attention_rows")
    return out, lse


def attention_rows_backward_workspace_bytes(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1, right: int = -1) -> int:
    """The workspace attention_rows_backward takes for these arguments."""
    p = _attention_params(q, k, v, cu_q, cu_k, left, right, scale)[0]
    n = int(load_library().nxg_attention_rows_backward_workspace_bytes(ctypes.byref(p)))
    _check(-n if n < 0 else 0, "attention_rows_backward_workspace_bytes")
    return n


def attention_rows_backward(dout, q, k, v, out, lse, cu_q, cu_k=None, scale: Optional[float] = None, left: int = -1,
                            right: int = -1, dq=None, dk=None, dv=None, workspace=None, stream=None):
    """The gradients of attention_rows: (dq, dk, dv), from dout, its inputs and what it returned (out, lse).
    Rows of no document are left as they were. workspace: None (made for the call) or a uint8 device tensor of
    attention_rows_backward_workspace_bytes."""
    torch = _torch()
    L = load_library()
    p, (qr, kr, vr), cu_q, cu_k = _attention_params(q, k, v, cu_q, cu_k, left, right, scale)
    T, H, D = q.shape
    gr, orows = _head_rows(dout, "dout", q, q.shape), _head_rows(out, "out", q, q.shape)
    _on_current_device(lse, "lse")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (T, H) or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 tensor [{T}][{H}]")
    made = []
    for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        made.append(torch.empty(like.shape, dtype=q.dtype, device=q.device) if t is None else t)
        if t is not None:
            _head_rows(t, name, q, like.shape)
    dqr, dkr, dvr = (_Rows(t.data_ptr(), t.stride(0), t.stride(1)) for t in made)
    n = int(L.nxg_attention_rows_backward_workspace_bytes(ctypes.byref(p)))
    _check(-n if n < 0 else 0, "attention_rows_backward")
    ws = _workspace(workspace, n, q.device)
    _order_on(stream, cu_q, cu_k, *made, ws)
    _check(L.nxg_attention_rows_backward(ctypes.byref(p), ctypes.byref(gr), ctypes.byref(qr), ctypes.byref(kr), ctypes.byref(vr),
                                         ctypes.byref(orows), lse.data_ptr(), ctypes.byref(dqr), ctypes.byref(dkr),
                                         ctypes.byref(dvr), ws.data_ptr(), ws.numel(), _stream_ptr(stream)),
           "attention_rows_backward")
    return tuple(made)
