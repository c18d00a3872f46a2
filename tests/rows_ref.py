"""The row operators of include/nxg_rows.h in 64 bits, from their definitions, with what their roundings
can make of a result at most: every function returns pairs (value, bound).

The bounds count, for a type whose roundings are off by at most u = eps / 2 of a value (and half of
its smallest step below its normal range):
  - the result's own rounding, u |result|;
  - the roundings of what is carried in that type between two products (attention's P and dS), each
    u of a term, so u times the sum of the terms' sizes;
  - fp32 sums of n terms, n 2^-24 times the sum of their sizes.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24
# An exponential, or a product of a matrix instruction, below fp32's normal numbers may be taken as 0: a
# weight or term is then off by less than the smallest normal number.
TINY = 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least_step(dtype):
    """Half the distance of the type's smallest numbers."""
    return {torch.float64: 0.0, torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]


def check(name, got, ref, bound):
    got, ref, bound = got.double().cpu(), ref.cpu(), bound.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], ref[inf]), f"{name}: infinities in other places"
    ok = torch.isfinite(ref)
    d = (got - ref).abs()
    bad = ok & ~(d <= bound)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values are off by more than their bound, the first at {at}: "
                             f"{got[at].item()} for {ref[at].item()} (bound {bound[at].item()})")


def rope(x, freq, pos, layout, mscale, inverse):
    """x [T][H][D], freq [n / 2] float64, pos [T]: ints."""
    u, X = half_step(x.dtype), x.double()
    n = 2 * freq.numel()
    angle = pos.double()[:, None] * freq.double()[None, :]
    c, s = torch.cos(angle)[:, None, :] * mscale, torch.sin(angle)[:, None, :] * mscale
    if inverse:
        s = -s
    ia = torch.arange(n // 2, device=x.device) * (1 if layout == "half" else 2)
    ib = ia + (n // 2 if layout == "half" else 1)
    y, slack = X.clone(), torch.zeros_like(X)
    a, b = X[..., ia], X[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    # the turn within a turn as fp32 (2^-26 of one), sin and cos (2 steps), the products and the sum; the
    # angle's own rounding in 64 bits, here and there
    e = 2 * math.pi * 2.0 ** -26 + 2.0 ** -22 + 6 * F32 + angle.abs()[:, None, :] * 2.0 ** -51
    slack[..., ia] = slack[..., ib] = (a.abs() + b.abs()) * abs(mscale) * e
    bound = slack + u * y.abs() * (1 + 1e-3) + least_step(x.dtype)
    bound[..., n:] = 0
    return y, bound


def layer_norm(x, w, b, eps):
    """((y, bound), (mean, bound), (rstd, bound))."""
    u, X, C = half_step(x.dtype), x.double(), x.shape[1]
    W = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    B = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    var, mean = torch.var_mean(X, 1, correction=0)
    rstd = (var + eps) ** -0.5
    k = (64 + C / 256) * F32                          # a thread's terms one after another, then a tree
    em = k * X.abs().mean(1)
    er = em * rstd + em * em * rstd * rstd + k + 8 * F32          # of rstd, relative
    h = (X - mean[:, None]) * rstd[:, None]
    y = h * W + B
    by = (em[:, None] * rstd[:, None] + h.abs() * (er[:, None] + 4 * F32)) * W.abs() + 2 * F32 * (y.abs() + B.abs()) + u * y.abs() * (1 + 1e-3)
    return (y, by + least_step(x.dtype)), (mean, em + F32 * mean.abs()), (rstd, rstd * er * (1 + 1e-3))


def layer_norm_back(dy, x, mean, rstd, w):
    """((dx, bound), (dw, bound), (db, bound)) with the forward call's mean and rstd."""
    u, C, T = half_step(x.dtype), x.shape[1], x.shape[0]
    G, W = dy.double(), torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    uw = half_step(torch.float32 if w is None else w.dtype)
    r = rstd.double()[:, None]
    h = (x.double() - mean.double()[:, None]) * r
    g = G * W
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - mg - h * mgh)
    k = (70 + C / 256) * F32
    slack = r * (8 * F32 * (g.abs() + mg.abs() + (h * mgh).abs()) + k * (g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)))
    kt = (128 + T / 256) * F32
    dw, db = (G * h).sum(0), G.sum(0)
    return ((dx, slack + u * dx.abs() * (1 + 1e-3) + least_step(x.dtype)),
            (dw, kt * (G * h).abs().sum(0) + uw * dw.abs() * (1 + 1e-3) + least_step(x.dtype)),
            (db, kt * G.abs().sum(0) + uw * db.abs() * (1 + 1e-3) + least_step(x.dtype)))


def window(n, m, left, right, device):
    """[n][m]: does query i see key j."""
    d = torch.arange(m, device=device)[None, :] - (torch.arange(n, device=device)[:, None] + (m - n))
    seen = torch.ones(n, m, dtype=torch.bool, device=device)
    if left >= 0:
        seen &= d >= -left
    if right >= 0:
        seen &= d <= right
    return seen


def attention(q, k, v, cu_q, cu_k, scale, left, right, dout=None):
    """{"out", "lse", "dq", "dk", "dv"}: (value, bound), over the rows of the documents (others: NaN in
    value and bound). Sums run over the pairs that see each other and no others."""
    u, dt = half_step(q.dtype), q.dtype
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    dev = q.device
    new = lambda t: torch.full(t.shape, math.nan, dtype=torch.float64, device=dev)  # noqa: E731
    res = {"out": (new(q), new(q)), "lse": (new(q[..., 0]), new(q[..., 0]))}
    if dout is not None:
        res.update({"dq": (new(q), new(q)), "dk": (new(k), new(k)), "dv": (new(v), new(v))})
        # fp16: dS is carried times 2^(15 - e), 2^e past twice the largest norms' product
        fin = lambda t: torch.nan_to_num(t.double(), 0.0, 0.0, 0.0)  # noqa: E731
        top = 2 * float(fin(dout).norm(dim=2).max()) * float(fin(v).norm(dim=2).max()) if q.numel() and v.numel() else 0.0
        ds_step = 0.0 if dt == torch.bfloat16 else 2.0 ** -25 * 2.0 ** (math.frexp(top * 1.01)[1] - 15) if top > 0 else 2.0 ** -25
    for a, b, c, d in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        a, b, c, d = int(a), int(b), int(c), int(d)
        seen = window(b - a, d - c, left, right, dev)
        for g in range(G):
            K, V = k[c:d, g].double(), v[c:d, g].double()
            if dout is not None:
                sums = {x: torch.zeros(d - c, D, dtype=torch.float64, device=dev) for x in ("dk", "dv", "bk", "bv")}
            for h in range(g * (H // G), (g + 1) * (H // G)):
                Q = q[a:b, h].double()
                # products over the seen pairs alone: what the others hold has no part
                S = torch.where(seen, (Q @ K.t()) * scale, -math.inf)
                size = float((Q.abs().amax(1, keepdim=True) if Q.numel() else Q.new_zeros(1)).max()) if Q.numel() else 0.0
                es = ((D + 8) * F32 * scale * (Q.abs() @ K.abs().t())).nan_to_num(0, 0, 0) if size else torch.zeros_like(S)
                es = torch.where(seen, es, torch.zeros_like(es)).amax(1, keepdim=True) if d > c else Q.new_zeros(b - a, 1)
                smax = torch.where(seen, S.abs(), torch.zeros_like(S)).nan_to_num(0, 0, 0).amax(1, keepdim=True) if d > c else Q.new_zeros(b - a, 1)
                ep = 2 * es + 8 * F32 * (smax + 1) + (d - c) * F32              # of a weight, relative
                empty = ~seen.any(1)
                L = torch.where(empty, -math.inf, torch.logsumexp(S, 1)) if d > c else Q.new_full((b - a,), -math.inf)
                P = torch.exp(S - L[:, None])
                P = torch.where(seen, P, torch.zeros_like(P))
                O, bo = _product(P, V, seen, dt)
                bo = (u * 1.01 + 4 * ep) * bo + u * O.abs() + ((0 if dt == torch.bfloat16 else 2.0 ** -24) + TINY) * (_product(seen.double(), V, seen, dt)[1] + (d - c)) + least_step(dt)
                O = torch.where(empty[:, None], torch.zeros_like(O), O)
                res["out"][0][a:b, h], res["out"][1][a:b, h] = O, torch.where(empty[:, None], torch.zeros_like(bo), bo)
                res["lse"][0][a:b, h] = L
                res["lse"][1][a:b, h] = torch.where(empty, torch.zeros_like(L), (2 * ep[:, 0] + 4 * F32 * (L.abs() + 1)))
                if dout is None:
                    continue
                dO = dout[a:b, h].double()
                dV, bv = _product(P.t(), dO, seen.t(), dt)
                sums["dv"] += dV
                sums["bv"] += (u * 1.01 + 4 * float(ep.max() if ep.numel() else 0) + 2.0 ** -20) * bv + ((0 if dt == torch.bfloat16 else 2.0 ** -39) + TINY) * (_product(seen.t().double(), dO, seen.t(), dt)[1] + (b - a))
                dP = torch.where(seen, dO @ V.t(), torch.zeros_like(P))
                delta = (dO * O).sum(1, keepdim=True)
                e_delta = (dO.abs() * bo).sum(1, keepdim=True) + (D + 4) * F32 * (dO.abs() * O.abs()).sum(1, keepdim=True)
                dS = torch.where(seen, P * (dP - delta), torch.zeros_like(P))
                e_dp = torch.where(seen, (D + 4) * F32 * (dO.abs() @ V.abs().t()), torch.zeros_like(P))
                e_ds = torch.where(seen, P * (e_delta + e_dp) * (1 + 4 * ep) + dS.abs() * (u * 1.01 + 4 * ep + 4 * F32) + P * delta.abs() * 4 * F32 + ds_step
                                   + TINY * (dP.abs() + delta.abs() + 1),
                                   torch.zeros_like(P))
                dQ, _ = _product(dS, K, seen, dt)
                bq = _product(e_ds + (d - c) * F32 * dS.abs(), K, seen, dt)[1] + TINY * (d - c)
                res["dq"][0][a:b, h] = dQ * scale
                res["dq"][1][a:b, h] = bq * scale + u * 1.01 * (dQ * scale).abs() + least_step(dt)
                dK, _ = _product(dS.t(), Q, seen.t(), dt)
                sums["dk"] += dK * scale
                sums["bk"] += _product((e_ds + (b - a) * F32 * dS.abs()).t(), Q, seen.t(), dt)[1] * scale + TINY * (b - a)
            if dout is not None:
                res["dk"][0][c:d, g], res["dk"][1][c:d, g] = sums["dk"], sums["bk"] * 1.01 + u * 1.01 * sums["dk"].abs() + least_step(dt)
                res["dv"][0][c:d, g], res["dv"][1][c:d, g] = sums["dv"], sums["bv"] * 1.01 + u * 1.01 * sums["dv"].abs() + least_step(dt)
    return res


def _product(w, x, seen, dt):
    """(w x, |w| |x|) where a pair that is not seen adds nothing, whatever x holds there."""
    if bool(torch.isfinite(x).all()) or w.shape[1] == 0:
        return w @ x, w.abs() @ x.abs()
    t = torch.where(seen[:, :, None], w[:, :, None] * x[None, :, :], torch.zeros((), dtype=torch.float64, device=x.device))
    return t.sum(1), t.abs().sum(1)
