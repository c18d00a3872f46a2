"""The row operators of adapter fine-tuning (include/nxg_rows.h) in 64 bits, from their definitions, with what their roundings can
make of a result at most: pairs (value, bound), as rows_ref.py counts them.

Beside 16-bit rows, adapter_rows carries s and g as the sum of two bf16 values between its products. A bf16 rounding is off by
2^-8 of a value at most, so the sum by 2^-16; fp16 rows, which are such a sum exactly, leave the product of both second
parts out: 2^-16 more.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from rows_ref import F32, TINY, half_step, least_step


def carried(dtype):
    """How far a value of s or g is off in the next product, relative."""
    return {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -15}[dtype]


# --- norms of queries and keys, and their rotation -----------------------------------------------

def _pairs(n, layout, device):
    ia = torch.arange(n // 2, device=device) * (1 if layout == "half" else 2)
    return ia, ia + (n // 2 if layout == "half" else 1)


def _turned(x, ex, freq, pos, layout, mscale, inverse):
    """x [T][H][D] (float64, off by ex) with its pairs turned, and what it is off by."""
    angle = pos.double()[:, None] * freq.double()[None, :]
    c, s = torch.cos(angle)[:, None, :] * mscale, torch.sin(angle)[:, None, :] * mscale * (-1 if inverse else 1)
    ia, ib = _pairs(2 * freq.numel(), layout, x.device)
    y, ey = x.clone(), ex.clone()
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    # the turn within a turn as fp32, sin and cos, the products and the sum; the angle's rounding in 64 bits
    e = 2 * math.pi * 2.0 ** -26 + 2.0 ** -22 + 6 * F32 + angle.abs()[:, None, :] * 2.0 ** -51
    ey[..., ia] = ey[..., ib] = ((a.abs() + b.abs()) * e + (ex[..., ia] + ex[..., ib])) * abs(mscale)
    return y, ey


# a sum of a head's values: up to 16 in a lane, 6 steps over lanes; the mean, eps, root and quotient
HEAD_SUM = 24 * F32
RSTD = 16 * F32


def qk_norm_rope(x, w, freq, pos, layout, mscale, eps):
    u, X = half_step(x.dtype), x.double()
    rstd = (X.square().mean(2, keepdim=True) + eps) ** -0.5
    h = X * rstd * w.double()
    y, ey = _turned(h, h.abs() * (RSTD + 3 * F32), freq, pos, layout, mscale, False)
    return y, ey + u * y.abs() * (1 + 1e-3) + least_step(x.dtype)


def qk_norm_rope_back(dy, x, w, freq, pos, layout, mscale, eps):
    """((dx, bound), (dw, bound))."""
    X, W = x.double(), w.double()
    G, eg = _turned(dy.double(), torch.zeros_like(X), freq, pos, layout, mscale, True)
    rstd = (X.square().mean(2, keepdim=True) + eps) ** -0.5
    h = X * rstd
    g = G * W
    e = eg * W.abs() + 2 * F32 * g.abs()
    m = (g * h).mean(2, keepdim=True)
    em = (e * h.abs()).mean(2, keepdim=True) + (HEAD_SUM + RSTD + 4 * F32) * (g * h).abs().mean(2, keepdim=True)
    dx = rstd * (g - h * m)
    slack = rstd * (e + h.abs() * em + (RSTD + 6 * F32) * (h * m).abs() + (RSTD + 4 * F32) * (g.abs() + (h * m).abs()))
    n = x.shape[0] * x.shape[1]
    dw = (G * h).sum((0, 1))
    bw = (eg * h.abs() + (RSTD + 3 * F32) * (G * h).abs()).sum((0, 1)) + (256 + n / 64) * F32 * (G * h).abs().sum((0, 1))
    return ((dx, slack * (1 + 1e-3) + half_step(x.dtype) * dx.abs() * (1 + 1e-3) + least_step(x.dtype)),
            (dw, bw * (1 + 1e-3) + half_step(w.dtype) * dw.abs() * (1 + 1e-3) + least_step(w.dtype)))


# --- dropout -------------------------------------------------------------------------------------

def philox(counter, key):
    """Philox 4x32-10 of Salmon, Moraes, Dror and Shaw (2011): counter [..., 4] and key (2) of 32-bit words."""
    c = [np.asarray(counter[..., i]) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, half = np.uint64(2 ** 32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, -1)


def kept(T, C, p, seed, offset):
    """bool [T][C]."""
    groups = (C + 7) // 8
    c = np.zeros((T, groups, 4), np.uint64)
    c[..., 0], c[..., 1] = np.arange(groups), np.arange(T)[:, None]
    c[..., 2], c[..., 3] = offset % 2 ** 32, offset // 2 ** 32 % 2 ** 32
    w = philox(c, (seed % 2 ** 32, seed // 2 ** 32))
    bits = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(T, groups * 8)[:, :C]
    return bits >= round(p * 65536)


def dropout(x, residual, p, seed, offset):
    u = half_step(x.dtype)
    keep = torch.from_numpy(kept(*x.shape, p, seed, offset)).to(x.device)
    v = torch.where(keep, x.double() * (65536 / (65536 - round(p * 65536))), 0.0)
    r = torch.zeros_like(v) if residual is None else residual.double()
    y = v + r
    return y, torch.where(keep, 3 * F32 * (v.abs() + r.abs()) + u * y.abs() * (1 + 1e-3) + least_step(x.dtype), 0.0)


# --- low-rank adapters -----------------------------------------------------------------------------

def _documents(cu, ids, n):
    """(rows, adapter or None) of every document."""
    for d in range(len(ids)):
        i = int(ids[d])
        yield slice(int(cu[d]), int(cu[d + 1])), (i if 0 <= i < n else None)


def adapter(x, a, b, cu, ids, scale, base):
    """((y, bound), (s, bound)); NaN (value and bound) in rows of no document."""
    X, A, B, u, dt = x.double(), a.double(), b.double(), half_step(x.dtype), x.dtype
    T, K, N, r = x.shape[0], x.shape[1], b.shape[1], a.shape[1]
    new = lambda n: torch.full((T, n), math.nan, dtype=torch.float64, device=x.device)  # noqa: E731
    y, by, s, bs = new(N), new(N), new(r), new(r)
    for rows, i in _documents(cu, ids, a.shape[0]):
        old = torch.zeros(rows.stop - rows.start, N, dtype=torch.float64, device=x.device) if base is None else base[rows].double()
        if i is None:
            y[rows], by[rows], s[rows], bs[rows] = old, 0.0, 0.0, 0.0
            continue
        S = X[rows] @ A[i].t()
        es = (K + 8) * F32 * (X[rows].abs() @ A[i].abs().t()) + TINY * K
        s[rows], bs[rows] = S, es
        d = scale * (S @ B[i].t())
        y[rows] = old + d
        e = abs(scale) * ((es + (carried(dt) + (r + 8) * F32) * S.abs() + TINY) @ B[i].abs().t() + TINY * r)
        by[rows] = e + 3 * F32 * (old.abs() + d.abs()) + u * y[rows].abs() * (1 + 1e-3) + least_step(dt)
    return (y, by), (s, bs)


def adapter_back(dy, x, a, b, s, cu, ids, scale, base):
    """((dx, bound), (da, bound), (db, bound)) with the forward call's s."""
    G0, X, A, B, dt = dy.double(), x.double(), a.double(), b.double(), x.dtype
    T, K, N, r = x.shape[0], x.shape[1], b.shape[1], a.shape[1]
    dx, bx = (torch.full((T, K), math.nan, dtype=torch.float64, device=x.device) for _ in range(2))
    da, ba = torch.zeros_like(A), torch.zeros_like(A)
    db, bb = torch.zeros_like(B), torch.zeros_like(B)
    for rows, i in _documents(cu, ids, a.shape[0]):
        old = torch.zeros(rows.stop - rows.start, K, dtype=torch.float64, device=x.device) if base is None else base[rows].double()
        if i is None:
            dx[rows], bx[rows] = old, 0.0
            continue
        g = scale * (G0[rows] @ B[i])
        eg = abs(scale) * ((N + 10) * F32 * (G0[rows].abs() @ B[i].abs()) + TINY * N)
        d = g @ A[i]
        dx[rows] = old + d
        e = (eg + (carried(dt) + (r + 8) * F32) * g.abs() + TINY) @ A[i].abs() + TINY * r
        bx[rows] = e + 3 * F32 * (old.abs() + d.abs()) + half_step(dt) * dx[rows].abs() * (1 + 1e-3) + least_step(dt)
        S = s[rows].double()
        da[i] += g.t() @ X[rows]
        ba[i] += (eg + (carried(dt) + (T + 16) * F32) * g.abs() + TINY).t() @ X[rows].abs() + TINY * T
        db[i] += scale * (G0[rows].t() @ S)
        bb[i] += abs(scale) * (G0[rows].abs().t() @ ((carried(dt) + (T + 16) * F32) * S.abs() + TINY) + TINY * T)
    uw = half_step(a.dtype)
    return ((dx, bx), (da, ba + uw * da.abs() * (1 + 1e-3) + least_step(a.dtype)), (db, bb + uw * db.abs() * (1 + 1e-3) + least_step(b.dtype)))
