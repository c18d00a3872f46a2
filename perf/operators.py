"""The floating-point row operators whose speed is measured, through the engine's public entry points.

Kinds of case ("op"):

  rope       rope_rows: rotary positions of packed documents
  norm       layer_norm_rows: the forward pass and what its gradient needs
  norm_back  layer_norm_rows_backward: gradients of the rows, the weight and the bias
  attention  attention_rows: grouped-query attention of packed documents, any window
  train      attention_rows, then attention_rows_backward: a training step's attention

Sizes are those of the 213M-parameter encoder (n_embd 1,024, FFN 2,304, 16 query and 8 KV heads
of 64, sliding window 256) at the lengths that the benchmark, the tests and the published timings
use; heads of 128 and the head ratios of `draw` are generic.

With `own` false, `run` computes the same from elementary torch operations in 32 bits (angles
and sums over all rows in 64), rounded once at the end.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

C, INTER, HEADS, KV_HEADS, HEAD_DIM = 1024, 2304, 16, 8, 64
BAND = 128                                   # |i - j| of the sliding window of 256
EPS = 1e-5
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# lengths of a mixed batch: 32 documents of 16 to 2,048 tokens (numpy's default_rng(1))
DOCS32 = " ".join(str(n) for n in np.random.default_rng(1).integers(16, 2048, 32, endpoint=True))
SHORT = "23 7 61 34"                         # a request of a few short texts
CHUNK = 1 << 29                              # scores that the plain form holds at a time


def _nxg():
    """The engine package, whose directory name is not an identifier."""
    name = "nexterabert_cpp_amd"
    if name not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "nexterabert.cpp_amd"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _rope_case(lengths, dtype, heads=HEADS + KV_HEADS, dim=HEAD_DIM, rot=HEAD_DIM, layout="half", scaling="none",
               factor=1.0, train_len=0, inverse=False, fused=True):
    return {"op": "rope", "lengths": lengths, "dtype": dtype, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "base": 100000.0, "scaling": scaling, "factor": factor, "train_len": train_len, "inverse": inverse,
            "fused": fused}


def _norm_case(op, rows, dtype, cols=C, wtype="fp32"):
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "wtype": wtype}


def _attention_case(op, lengths, dtype, left=-1, right=-1, keys="", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM,
                    layout="rows"):
    return {"op": op, "lengths": lengths, "keys": keys, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "left": left, "right": right, "layout": layout}


def listed():
    return [
        # queries and keys of a few short texts inside their fused projection: a launch's latency
        {"name": "rope_125", **_rope_case(SHORT, "bf16")},
        # the longest document the published timings have, scaled past a trained length of 8,192,
        # half of each head turned, neighbouring pairs
        {"name": "rope_65536", **_rope_case("65536", "fp32", rot=32, layout="interleaved", scaling="by_parts",
                                            factor=8.0, train_len=8192)},
        # the output norm of a few short texts, and of the longest document
        {"name": "norm_125", **_norm_case("norm", 125, "fp32")},
        {"name": "norm_65536", **_norm_case("norm", 65536, "bf16")},
        # its gradients in a training step over a mixed batch (fp32 weights over 16-bit rows)
        {"name": "norm_back_32docs", **_norm_case("norm_back", sum(map(int, DOCS32.split())), "bf16")},
        # attention of a request of a few short texts: latency
        {"name": "attention_short", **_attention_case("attention", SHORT, "bf16")},
        # one new query per document over a mixed batch of documents: what reading K and V costs
        {"name": "attention_1query_32docs", **_attention_case("attention", " ".join(["1"] * 32), "bf16", keys=DOCS32)},
        # a causal prompt batch of mixed lengths
        {"name": "attention_causal_32docs", **_attention_case("attention", DOCS32, "bf16", right=0)},
        # the longest document, every key
        {"name": "attention_65536", **_attention_case("attention", "65536", "bf16")},
        # training: the sliding window over a batch of 8, full attention over the mixed batch (both
        # inside the fused projection's rows), and a long causal document with heads of 128
        {"name": "train_band_8x1024", **_attention_case("train", " ".join(["1024"] * 8), "bf16", left=BAND, right=BAND,
                                                        layout="fused")},
        {"name": "train_32docs", **_attention_case("train", DOCS32, "bf16", layout="fused")},
        {"name": "train_causal_8192", **_attention_case("train", "8192", "fp16", right=0, dim=128)},
    ]


# --- drawn cases -------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_lengths(rng, most, docs=32):
    """One document, several alike, or a mixed batch; at most `most` tokens in all."""
    shape = rng.choice(["one", "alike", "mixed", "mixed"])
    if shape == "one":
        return str(_log(rng, 1, most))
    if shape == "alike":
        n = rng.randint(2, min(16, docs))
        return " ".join([str(_log(rng, 1, max(2, min(2048, most // n))))] * n)
    out = []
    for _ in range(rng.randint(2, docs)):
        out.append(_log(rng, 1, 2048))
        if sum(out) > most:
            out[-1] = max(1, out[-1] - (sum(out) - most))
            break
    return " ".join(map(str, out))


def draw(rng):
    op = rng.choice(["rope", "norm", "norm_back", "attention", "attention", "train", "train"])
    if op == "rope":
        dim = rng.choice([64, 64, 128, 96, 80])
        rot = rng.choice([dim, dim, dim // 2])
        scaling = rng.choice(["none", "linear", "ntk", "by_parts"])
        return _rope_case(_draw_lengths(rng, 65536), rng.choice(["fp32", "fp16", "bf16"]), rng.choice([1, 8, 16, 24, 33]),
                          dim, rot, rng.choice(["half", "interleaved"]), scaling,
                          1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                          8192 if scaling == "by_parts" else 0, rng.random() < 0.3, rng.random() < 0.5)
    if op in ("norm", "norm_back"):
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        cols = rng.choice([C, C, INTER, 64, 320, 1023, 2560, 4096, _log(rng, 1, 8192)])
        return _norm_case(op, _log(rng, 1, min(65536, (1 << 27) // cols)), dtype, cols, rng.choice(["fp32", dtype]))
    dim = rng.choice([64, 64, 64, 128, 128, 32, 96, 80])
    heads, kv = rng.choice([(16, 8), (16, 8), (16, 16), (8, 1), (12, 4), (6, 2), (32, 4), (1, 1)])
    half = _log(rng, 1, 1024)
    left, right = rng.choice([(-1, -1), (-1, 0), (-1, 0), (half, half), (half, 0)])
    most = 65536 if left >= 0 else 16384 if op == "train" else 32768
    lengths = _draw_lengths(rng, most * 16 // max(16, heads) if left < 0 else most // 2)
    keys = ""
    kind = rng.random()
    n = len(lengths.split())
    if kind < 0.2:                                  # a few queries over many keys
        lengths = " ".join(str(rng.choice([1, 1, 1, 2, 5, 16])) for _ in range(n))
        keys = " ".join(str(_log(rng, 1, 65536 // n)) for _ in range(n))
    elif kind < 0.4:                                # another document's keys, some without any
        keys = " ".join(str(0 if rng.random() < 0.1 else _log(rng, 1, 2048)) for _ in range(n))
        if not any(map(int, keys.split())):
            keys = ""
    return _attention_case(op, lengths, rng.choice(["bf16", "bf16", "fp16"]), left, right, keys, heads, kv, dim,
                           "rows" if keys else rng.choice(["rows", "fused", "heads"]))


# --- what a case needs -------------------------------------------------------------------------

def _lengths(case, key="lengths"):
    return [int(n) for n in (case[key] or case["lengths"]).split()]


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _pairs(case):
    """(query, key) pairs of one head inside the window: key j of query i from
    i + n_k - n_q - left to i + n_k - n_q + right."""
    total = 0
    for n, m in zip(_lengths(case), _lengths(case, "keys")):
        i = np.arange(n, dtype=np.int64) + (m - n)
        lo = np.zeros(n, np.int64) if case["left"] < 0 else np.clip(i - case["left"], 0, m)
        hi = np.full(n, m, np.int64) if case["right"] < 0 else np.clip(i + case["right"] + 1, 0, m)
        total += int(np.maximum(hi - lo, 0).sum())
    return total


def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "rope":
        T = sum(_lengths(case))
        return {"bytes": 2 * size * T * case["heads"] * case["dim"], "flops": 3 * T * case["heads"] * case["rot"]}
    if case["op"] in ("norm", "norm_back"):
        n, cols = case["rows"] * case["cols"], case["cols"]
        wsize = {"fp32": 4, "fp16": 2, "bf16": 2}[case["wtype"]]
        if case["op"] == "norm":
            return {"bytes": 2 * size * n + 2 * wsize * cols + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * size * n + 3 * wsize * cols + 8 * case["rows"], "flops": 14 * n}
    T, D = sum(_lengths(case)), case["dim"]
    K = seen = 0                                                # keys, and those that some query sees
    for n, m in zip(_lengths(case), _lengths(case, "keys")):
        lo, hi = _span(case, n, m, 0, n)
        K, seen = K + m, seen + hi - lo
    q, row = T * case["heads"] * D * size, case["kv_heads"] * D * size
    one = 2 * D * case["heads"] * _pairs(case)                  # one product over the pairs
    if case["op"] == "attention":
        return {"bytes": 2 * q + 2 * seen * row, "flops": 2 * one}
    return {"bytes": 4 * q + 2 * (seen + K) * row, "flops": 7 * one}    # the scores once more in the backward pass


# --- inputs ------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _frequencies(case):
    """Radians per position of each pair and the factor on the result, as the scaling's formula
    gives them: positions / factor (linear), base * factor^(n / (n - 2)) (ntk), or each frequency
    between f / factor and f by its turns over the trained length, 1 to 32 (by_parts)."""
    n, base, factor = case["rot"], case["base"], case["factor"]
    if case["scaling"] == "ntk" and n > 2:
        base *= factor ** (n / (n - 2.0))
    f = float(base) ** (-2.0 * np.arange(n // 2) / n)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "by_parts":
        keep = np.clip((case["train_len"] * f / (2 * math.pi) - 1.0) / 31.0, 0.0, 1.0)
        return (1 - keep) * f / factor + keep * f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rope":
        lens = _lengths(case)
        T, H, D = sum(lens), case["heads"], case["dim"]
        # fused: the heads to turn are the first of a projection's rows, as many again (the values) behind
        s["x"] = _randn(g, dt, T, H + (H + 1) // 2, D)[:, :H] if case["fused"] else _randn(g, dt, T, H, D)
        s["cu"] = torch.from_numpy(_offsets(lens)).cuda()
        f, s["mscale"] = _frequencies(case)
        s["freq"] = torch.from_numpy(f).cuda()
        s["lens"] = lens
        return s
    if case["op"] in ("norm", "norm_back"):
        T, n, wt = case["rows"], case["cols"], DTYPES[case["wtype"]]
        # rows of a residual stream: of different sizes and off zero
        x = torch.randn(T, n, device="cuda", generator=g) * (0.5 + torch.rand(T, 1, device="cuda", generator=g))
        s["x"] = (x + 0.3 * torch.randn(1, n, device="cuda", generator=g)).to(dt)
        s["w"] = (0.8 + 0.4 * torch.rand(n, device="cuda", generator=g)).to(wt)
        s["b"] = (0.02 * torch.randn(n, device="cuda", generator=g)).to(wt)
        if case["op"] == "norm_back":
            s["dy"] = _randn(g, dt, T, n)
            x = s["x"].double()
            s["mean"] = x.mean(1).float()
            s["rstd"] = (x.var(1, unbiased=False) + EPS).rsqrt().float()
        return s
    lens, keys = _lengths(case), _lengths(case, "keys")
    T, K, H, G, D = sum(lens), sum(keys), case["heads"], case["kv_heads"], case["dim"]
    if case["layout"] == "fused":                   # one projection's rows
        rows = _randn(g, dt, T, H + 2 * G, D)
        s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + G], rows[:, H + G:]
    else:
        s["q"] = _randn(g, dt, T, H, D)
        if case["layout"] == "heads":               # one head's rows after another
            s["k"], s["v"] = (_randn(g, dt, G, K, D).transpose(0, 1) for _ in range(2))
        else:
            s["k"], s["v"] = (_randn(g, dt, K, G, D) for _ in range(2))
    if case["op"] == "train":
        s["dout"] = (0.1 * torch.randn(T, H, D, device="cuda", generator=g)).to(dt)
    s["cu_q"], s["cu_k"] = (torch.from_numpy(_offsets(n)).cuda() for n in (lens, keys))
    s["lens"], s["keys"] = lens, keys
    s["groups"] = _groups(case)                     # of use to the plain form
    return s


# --- one pass ----------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        nxg = _nxg()
        if case["op"] == "rope":
            return nxg.rope_rows(s["x"], s["freq"], s["cu"], layout=case["layout"], mscale=s["mscale"],
                                 inverse=case["inverse"])
        if case["op"] == "norm":
            return nxg.layer_norm_rows(s["x"], s["w"], s["b"], EPS)
        if case["op"] == "norm_back":
            return nxg.layer_norm_rows_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        window = {"left": case["left"], "right": case["right"], "scale": case["dim"] ** -0.5}
        out, lse = nxg.attention_rows(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], **window)
        if case["op"] == "attention":
            return out
        return (out,) + tuple(nxg.attention_rows_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["cu_q"],
                                                          s["cu_k"], **window))
    if case["op"] == "rope":
        return _plain_rope(s)
    if case["op"] == "norm":
        return _plain_norm(s)
    if case["op"] == "norm_back":
        return _plain_norm_back(s)
    return _plain_attention(s, case["op"] == "train")


# --- the plain forms: 32 bits, elementary operations ---------------------------------------------

def _plain_rope(s):
    case, x = s["case"], s["x"].float()
    pos = torch.arange(x.shape[0], device="cuda", dtype=torch.float64)
    starts = torch.repeat_interleave(s["cu"][:-1].double(), torch.diff(s["cu"]).long())
    angle = (pos - starts)[:, None] * s["freq"][None, :]
    cos = (torch.cos(angle) * s["mscale"]).float()[:, None, :]
    sin = (torch.sin(angle) * s["mscale"]).float()[:, None, :]
    if case["inverse"]:
        sin = -sin
    n, out = case["rot"], x.clone()
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        out[..., :n // 2] = a * cos - b * sin
        out[..., n // 2:n] = a * sin + b * cos
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        out[..., 0:n:2] = a * cos - b * sin
        out[..., 1:n:2] = a * sin + b * cos
    return out.to(s["x"].dtype)


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    y = d * rstd * s["w"].float() + s["b"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_back(s):
    dy, x = s["dy"].float(), s["x"].float()
    rstd = s["rstd"][:, None]
    h = (x - s["mean"][:, None]) * rstd
    g = dy * s["w"].float()
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    dw = (dy * h).sum(0, dtype=torch.float64)
    db = dy.sum(0, dtype=torch.float64)
    return dx.to(s["dy"].dtype), dw.to(s["w"].dtype), db.to(s["w"].dtype)


def _span(case, n, m, r, rows):
    """The keys that queries r .. r + rows of a document of n queries and m keys can see."""
    lo = 0 if case["left"] < 0 else max(0, r + m - n - case["left"])
    hi = m if case["right"] < 0 else min(m, r + rows + m - n + case["right"])
    return lo, max(lo, hi)


def _groups(case):
    """The documents in groups of like lengths, padded to one batch each: the rows of q and k of
    [document][position], row 0 behind a document's end, and the lengths."""
    lens, keys = np.array(_lengths(case)), np.array(_lengths(case, "keys"))
    t0, k0 = _offsets(lens)[:-1], _offsets(keys)[:-1]
    left, out = sorted(range(len(lens)), key=lambda d: (-keys[d], -lens[d])), []
    while left:
        n, m = lens[left].max(), keys[left[0]]
        most = max(1, CHUNK // (case["heads"] * max(1, n * m)))
        # all at once where they are few, else those of at least two thirds of the longest
        near = left if len(left) <= most else [d for d in left if 3 * keys[d] >= 2 * m][:most]
        left = [d for d in left if d not in near]
        n, m = lens[near].max(), keys[near].max()
        i, j = np.arange(n)[None, :], np.arange(m)[None, :]
        nd, md = lens[near][:, None], keys[near][:, None]
        pad = lambda start, at, size: torch.from_numpy(np.where(at < size, start[near][:, None] + at, 0)).cuda()  # noqa: E731
        # where each row of the documents is in the padded batch, one after another
        flat = lambda at, size: torch.from_numpy(np.flatnonzero(at < size)).cuda()  # noqa: E731
        dst = lambda start, at, size: torch.from_numpy((start[near][:, None] + at)[at < size]).cuda()  # noqa: E731
        out.append({"n": int(n), "m": int(m), "q": pad(t0, i, nd), "k": pad(k0, j, md),
                    "q_flat": flat(i, nd), "q_row": dst(t0, i, nd), "k_flat": flat(j, md), "k_row": dst(k0, j, md),
                    "nd": torch.from_numpy(nd).cuda(), "md": torch.from_numpy(md).cuda(), "alike": bool((nd == n).all() and (md == m).all())})
    return out


def _plain_attention(s, train):
    """Groups of documents as padded batches, all heads at a time, in pieces of the queries."""
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    H, G, D, R = case["heads"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    scale, left, right = case["dim"] ** -0.5, case["left"], case["right"]
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    if train:
        dq = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        dk, dv = (torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (k, v))
    for g in s["groups"]:
        B, n, m = g["nd"].shape[0], g["n"], g["m"]
        if m == 0:                                   # documents without keys
            out[g["q_row"]] = 0
            if train:
                dq[g["q_row"]] = 0
            continue
        heads = lambda t, rows: t[rows].float().transpose(1, 2).reshape(-1, rows.shape[1], D)       # noqa: E731
        kh, vh = heads(k, g["k"]), heads(v, g["k"])                                                  # B * G, m, D
        kt = kh.transpose(1, 2).contiguous()
        gq, y = (torch.empty(B, n, H, D, device="cuda") for _ in range(2))
        if train:
            vt = vh.transpose(1, 2).contiguous()
            gk, gv = torch.zeros_like(kh), torch.zeros_like(vh)
        step = max(1, CHUNK // (B * H * m))
        if left >= 0 and g["alike"]:                 # a piece sees few keys beside its own: pieces of that size
            step = min(step, max(256, left + max(right, 0)))
        for r in range(0, n, step):
            rows = min(step, n - r)
            lo, hi = _span(case, n, m, r, rows) if g["alike"] else (0, m)
            if lo >= hi:
                lo, hi = 0, m
            # B * G, R * rows, D: a KV head's queries one after another
            split = lambda t: t[g["q"][:, r:r + rows]].float().view(B, rows, G, R, D).permute(0, 2, 3, 1, 4).reshape(B * G, R * rows, D)  # noqa: E731
            join = lambda t: t.view(B, G, R, rows, D).permute(0, 3, 1, 2, 4).reshape(B, rows, H, D)   # noqa: E731
            qh = split(q)
            sc = torch.bmm(qh, kt[:, :, lo:hi].contiguous()).mul_(scale)
            if left >= 0 or right >= 0 or not g["alike"]:
                j = torch.arange(lo, hi, device="cuda")[None, None, :]
                at = torch.arange(r, r + rows, device="cuda")[None, :, None] + (g["md"] - g["nd"])[:, :, None]
                hide = j >= g["md"][:, :, None]
                if left >= 0:
                    hide = hide | (j < at - left)
                if right >= 0:
                    hide = hide | (j > at + right)
                sc.view(B, G * R, rows, hi - lo).masked_fill_(hide.expand(B, rows, hi - lo)[:, None], -math.inf)
            top = sc.amax(2, keepdim=True)
            p = sc.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
            total = p.sum(2, keepdim=True)
            p.div_(torch.where(total == 0, torch.ones_like(total), total))
            y[:, r:r + rows] = join(torch.bmm(p, vh[:, lo:hi].contiguous()))
            if not train:
                continue
            do = split(s["dout"])
            if not g["alike"]:                       # rows behind a document's end
                do.view(B, G * R, rows, D).mul_((torch.arange(r, r + rows, device="cuda") < g["nd"]).view(B, 1, rows, 1))
            gv[:, lo:hi] += torch.bmm(p.transpose(1, 2).contiguous(), do)
            dp = torch.bmm(do, vt[:, :, lo:hi].contiguous())
            ds = dp.sub_((dp * p).sum(2, keepdim=True)).mul_(p).mul_(scale)
            gq[:, r:r + rows] = join(torch.bmm(ds, kh[:, lo:hi].contiguous()))
            gk[:, lo:hi] += torch.bmm(ds.transpose(1, 2).contiguous(), qh)
        out[g["q_row"]] = y.view(B * n, H, D)[g["q_flat"]].to(q.dtype)
        if train:
            dq[g["q_row"]] = gq.view(B * n, H, D)[g["q_flat"]].to(q.dtype)
            rows = lambda t: t.view(B, G, m, D).transpose(1, 2).reshape(B * m, G, D)[g["k_flat"]]      # noqa: E731
            dk[g["k_row"]], dv[g["k_row"]] = rows(gk).to(k.dtype), rows(gv).to(v.dtype)
    return (out, dq, dk, dv) if train else out


# --- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s["x"].double(), s["lens"])
    if case["op"] == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS) ** -0.5
        return (x - mean[:, None]) * rstd[:, None] * s["w"].double() + s["b"].double(), mean, rstd
    if case["op"] == "norm_back":
        # by differentiation of the definition
        x, w = s["x"].double().requires_grad_(), s["w"].double().requires_grad_()
        b = torch.zeros_like(w).requires_grad_()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + b
        return torch.autograd.grad(y, (x, w, b), s["dy"].double())
    if case["op"] == "train" and _pairs(case) * case["heads"] > 3e9 * 4:
        return None
    return _exact_attention(case, s, case["op"] == "train")


def _exact_rope(case, x, lens):
    """Each pair as a complex number times mscale * e^(i * position * frequency)."""
    freq, mscale = _frequencies(case)
    pos = np.concatenate([np.arange(n) for n in lens])
    turn = torch.polar(torch.full((x.shape[0], 1, case["rot"] // 2), mscale, dtype=torch.float64, device="cuda"),
                       torch.from_numpy(pos[:, None, None] * freq).cuda() * (-1.0 if case["inverse"] else 1.0))
    n, head = case["rot"], x[..., :case["rot"]]
    if case["layout"] == "half":
        z = torch.complex(head[..., :n // 2], head[..., n // 2:]) * turn
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(*head.shape[:2], n // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(head.shape)
    return torch.cat([head, x[..., n:]], -1)


def _exact_attention(case, s, train):
    """Per document and query head; the gradients by differentiation."""
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    ratio = case["heads"] // case["kv_heads"]
    t0 = k0 = 0
    for n, m in zip(s["lens"], s["keys"]):
        step = max(1, (1 << 28) // max(1, m))
        for h in range(case["heads"]):
            kh = k[k0:k0 + m, h // ratio].contiguous().requires_grad_(train)
            vh = v[k0:k0 + m, h // ratio].contiguous().requires_grad_(train)
            for r in range(0, n, step):
                e = min(n, r + step)
                qh = q[t0 + r:t0 + e, h].contiguous().requires_grad_(train)
                sc = torch.mm(qh, kh.t()) * (case["dim"] ** -0.5)
                d = torch.arange(m, device="cuda") - (torch.arange(r, e, device="cuda") + m - n)[:, None]
                seen = torch.ones_like(d, dtype=torch.bool)
                if case["left"] >= 0:
                    seen = seen & (d >= -case["left"])
                if case["right"] >= 0:
                    seen = seen & (d <= case["right"])
                some = seen.any(1)
                if not bool(some.any()):
                    continue
                w = torch.softmax(sc[some].masked_fill(~seen[some], -math.inf), 1)
                y = torch.mm(w, vh)
                rows = torch.arange(t0 + r, t0 + e, device="cuda")[some]
                out[rows, h] = y.detach()
                if train:
                    a, b, c = torch.autograd.grad(y, (qh, kh, vh), s["dout"][rows, h].double())
                    dq[t0 + r:t0 + e, h] = a
                    dk[k0:k0 + m, h // ratio] += b
                    dv[k0:k0 + m, h // ratio] += c
        t0, k0 = t0 + n, k0 + m
    return (out, dq, dk, dv) if train else out
