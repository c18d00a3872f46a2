"""The row operators of adapter fine-tuning whose speed is measured, through the engine's public entry points.

Kinds of case ("op"):

  qk             qk_norm_rope_rows: the norms of queries and keys for each head, then the rotation
  qk_back        qk_norm_rope_rows_backward: gradients of the rows and of both norms' weights
  dropout        dropout_rows: a counter-based mask, with or without a residual
  adapter        adapter_rows: each document's own low-rank adapter beside a shared projection
  adapter_back   adapter_rows_backward: gradients of the rows and of every adapter
  adapter_train  adapter_rows, then adapter_rows_backward: a training step's adapters

Sizes are those of the 213M-parameter encoder (n_embd 1,024, FFN 2,304, 16 query and 8 KV heads of 64) at
the lengths that the benchmark, the tests and the published timings use; heads of 128, ranks and numbers of
adapters are generic.

With `own` false, `run` computes the same from elementary torch operations in 32 bits (angles and the
norm weights' sums in 64), rounded once at the end.
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
EPS = 1e-6
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
# lengths of a mixed batch: 32 documents of 16 to 2,048 tokens (numpy's default_rng(1))
DOCS32 = " ".join(str(n) for n in np.random.default_rng(1).integers(16, 2048, 32, endpoint=True))
SHORT = "23 7 61 34"                         # a request of a few short texts


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


def _qk_case(op, lengths, dtype, wtype="fp32", heads=HEADS, kv_heads=KV_HEADS, dim=HEAD_DIM, rot=HEAD_DIM, layout="half", fused=True):
    return {"op": op, "lengths": lengths, "dtype": dtype, "wtype": wtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "layout": layout, "base": 100000.0, "fused": fused}


def _dropout_case(rows, dtype, cols=C, p=0.1, residual=True, rng=20240229, offset=7):
    return {"op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "residual": residual, "rng": rng, "offset": offset}


def _adapter_case(op, lengths, dtype, wtype, ids, n, rank=16, n_in=C, n_out=C, base=True):
    """ids: each document's adapter of n, -1 for none."""
    return {"op": op, "lengths": lengths, "dtype": dtype, "wtype": wtype, "ids": ids, "n": n, "rank": rank, "n_in": n_in, "n_out": n_out,
            "base": base}


def _text(numbers):
    return " ".join(map(str, numbers))


def listed():
    return [
        # queries and keys of a few short texts inside their fused projection: a launch's latency
        {"name": "qk_125", **_qk_case("qk", SHORT, "bf16")},
        # a training step's mixed batch inside the fused projection, forward and back
        {"name": "qk_32docs", **_qk_case("qk", DOCS32, "bf16")},
        {"name": "qk_back_32docs", **_qk_case("qk_back", DOCS32, "bf16")},
        # the longest document the published timings have: heads of 128 of which half is turned, neighbouring pairs
        {"name": "qk_65536", **_qk_case("qk", "65536", "fp16", "fp16", dim=128, rot=64, layout="interleaved", fused=False)},
        # the dropout before a block's residual, in the engine's own fp32 rows: a few short texts (latency), and a mixed batch
        {"name": "dropout_125", **_dropout_case(125, "fp32")},
        {"name": "dropout_32docs", **_dropout_case(sum(map(int, DOCS32.split())), "bf16")},
        # the gradient of an FFN's inner dropout over the longest document
        {"name": "dropout_65536", **_dropout_case(65536, "bf16", INTER, residual=False)},
        # serving: one row of one request, fp32 rows as the int8 linears leave them; 64 requests of one row, an adapter each
        {"name": "adapter_1row", **_adapter_case("adapter", "1", "fp32", "bf16", "2", 4, n_out=INTER)},
        {"name": "adapter_64x1", **_adapter_case("adapter", _text([1] * 64), "bf16", "bf16", _text((7 * i) % 64 for i in range(64)), 64)},
        # a mixed batch of requests with 8 adapters, every ninth document without, beside an int8 linear's fp32 rows
        {"name": "adapter_32docs", **_adapter_case("adapter", DOCS32, "fp32", "bf16", _text(i % 9 - 1 for i in range(32)), 8)},
        # training: the gradients over the mixed batch with four tasks' adapters, and one adapter of rank 64 over the longest document
        {"name": "adapter_back_32docs", **_adapter_case("adapter_back", DOCS32, "bf16", "bf16", _text(i % 4 for i in range(32)), 4)},
        {"name": "adapter_train_65536", **_adapter_case("adapter_train", "65536", "bf16", "bf16", "0", 1, rank=64, n_out=INTER)},
    ]


# --- drawn cases -------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_lengths(rng, most, docs=32):
    """One document, several alike, or a mixed batch; at most `most` tokens in all."""
    shape = rng.choice(["one", "alike", "mixed", "mixed"])
    if shape == "one":
        return [_log(rng, 1, most)]
    if shape == "alike":
        n = rng.randint(2, min(16, docs))
        return [_log(rng, 1, max(2, min(2048, most // n)))] * n
    out = []
    for _ in range(rng.randint(2, docs)):
        out.append(_log(rng, 1, 2048))
        if sum(out) > most:
            out[-1] = max(1, out[-1] - (sum(out) - most))
            break
    return out


def draw(rng):
    op = rng.choice(["qk", "qk_back", "dropout", "adapter", "adapter", "adapter_back", "adapter_train"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op in ("qk", "qk_back"):
        dim = rng.choice([64, 64, 128, 96, 80, 32])
        heads, kv = rng.choice([(16, 8), (16, 8), (16, 16), (8, 1), (12, 4), (32, 4), (1, 1)])
        most = min(65536, (1 << 27) // ((heads + kv) * dim)) // (2 if op == "qk_back" else 1)
        return _qk_case(op, _text(_draw_lengths(rng, most)), dtype, rng.choice(["fp32", dtype]), heads, kv, dim,
                        rng.choice([dim, dim, dim // 2]), rng.choice(["half", "interleaved"]), rng.random() < 0.5)
    if op == "dropout":
        cols = rng.choice([C, C, INTER, 64, 1023, 4096, _log(rng, 1, 8192)])
        return _dropout_case(_log(rng, 1, min(65536, (1 << 26) // cols)), dtype, cols, rng.choice([0.05, 0.1, 0.2, 0.5, 0.9]),
                             rng.random() < 0.6, rng.randrange(1 << 62), rng.randrange(1 << 40))
    n_in, n_out = rng.choice([(C, C), (C, INTER), (INTER, C), (C, HEADS * HEAD_DIM + 2 * KV_HEADS * HEAD_DIM), (320, 1000), (1023, 65)])
    rank = rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 64)])
    n = rng.choice([1, 1, 2, 4, 8, 64])
    most = max(64, (65536 // 4) * 16 // max(16, rank))
    if op == "adapter" and rng.random() < 0.4:          # requests of one row each
        lens = [1] * rng.randint(1, 256)
    else:
        lens = _draw_lengths(rng, most)
    ids = [-1 if rng.random() < 0.05 and len(lens) > 1 else rng.randrange(n) for _ in lens]
    return _adapter_case(op, _text(lens), dtype, rng.choice(["fp32", "bf16", "fp16"]) if dtype == "fp32" else dtype, _text(ids), n, rank,
                         n_in, n_out, rng.random() < 0.7)


# --- what a case needs -------------------------------------------------------------------------

def _numbers(case, key="lengths"):
    return [int(n) for n in case[key].split()]


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] in ("qk", "qk_back"):
        n = sum(_numbers(case)) * (case["heads"] + case["kv_heads"])
        w = 2 * case["dim"] * SIZES[case["wtype"]]
        if case["op"] == "qk":
            return {"bytes": 2 * size * n * case["dim"] + w, "flops": n * (4 * case["dim"] + 3 * case["rot"])}
        return {"bytes": 3 * size * n * case["dim"] + 2 * w, "flops": n * (10 * case["dim"] + 3 * case["rot"])}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": size * n * (3 if case["residual"] else 2), "flops": 2 * n}
    lens, ids = _numbers(case), _numbers(case, "ids")
    wsize, base = SIZES[case["wtype"]], 1 if case["base"] else 0
    T, mine = sum(lens), sum(n for n, i in zip(lens, ids) if i >= 0)
    weights = case["rank"] * (case["n_in"] + case["n_out"]) * wsize
    used = len({i for n, i in zip(lens, ids) if i >= 0 and n > 0}) * weights
    fwd = size * (mine * case["n_in"] + T * case["n_out"] * (1 + base)) + used + 4 * T * case["rank"]
    back = size * (mine * (case["n_in"] + case["n_out"]) + T * case["n_in"] * (1 + base)) + used + case["n"] * weights + 4 * T * case["rank"]
    one = 2 * mine * case["rank"] * (case["n_in"] + case["n_out"])
    return {"bytes": (fwd if case["op"] != "adapter_back" else 0) + (back if case["op"] != "adapter" else 0),
            "flops": one * {"adapter": 1, "adapter_back": 2, "adapter_train": 3}[case["op"]]}


# --- inputs ------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _frequencies(case):
    n = case["rot"]
    return float(case["base"]) ** (-2.0 * np.arange(n // 2) / n)


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("qk", "qk_back"):
        lens = _numbers(case)
        T, H, G, D, wt = sum(lens), case["heads"], case["kv_heads"], case["dim"], DTYPES[case["wtype"]]

        def heads():                                # fused: queries and keys are the first of a projection's rows, the values behind
            if case["fused"]:
                rows = _randn(g, dt, T, H + 2 * G, D)
                return rows[:, :H], rows[:, H:H + G]
            return _randn(g, dt, T, H, D), _randn(g, dt, T, G, D)
        s["q"], s["k"] = heads()
        s["wq"], s["wk"] = ((0.8 + 0.4 * torch.rand(D, device="cuda", generator=g)).to(wt) for _ in range(2))
        if case["op"] == "qk_back":
            s["dq_out"], s["dk_out"] = (0.1 * _randn(g, torch.float32, T, n, D) for n in (H, G))
            s["dq_out"], s["dk_out"] = s["dq_out"].to(dt), s["dk_out"].to(dt)
        s["cu"] = torch.from_numpy(_offsets(lens)).cuda()
        s["freq"] = torch.from_numpy(_frequencies(case)).cuda()
        s["lens"] = lens
        return s
    if case["op"] == "dropout":
        s["x"] = _randn(g, dt, case["rows"], case["cols"])
        s["residual"] = _randn(g, dt, case["rows"], case["cols"]) if case["residual"] else None
        return s
    lens, ids, n, r, wt = _numbers(case), _numbers(case, "ids"), case["n"], case["rank"], DTYPES[case["wtype"]]
    T, K, N = sum(lens), case["n_in"], case["n_out"]
    s["x"] = _randn(g, dt, T, K)
    s["a"] = (torch.randn(n, r, K, device="cuda", generator=g) * K ** -0.5).to(wt)
    s["b"] = (torch.randn(n, N, r, device="cuda", generator=g) * 0.3 * r ** -0.5).to(wt)
    s["cu"] = torch.from_numpy(_offsets(lens)).cuda()
    s["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
    s["scale"] = 2.0
    if case["op"] != "adapter_back":
        s["base"] = _randn(g, dt, T, N) if case["base"] else None
    if case["op"] != "adapter":
        s["dy"] = (0.1 * torch.randn(T, N, device="cuda", generator=g)).to(dt)
        s["dx_base"] = (0.1 * torch.randn(T, K, device="cuda", generator=g)).to(dt) if case["base"] else None
    s["rows"] = _rows_of(lens, ids)                 # of use to the plain form
    if case["op"] == "adapter_back":                # what the forward call left
        s["s"] = torch.zeros(T, r, device="cuda")
        for i, rows in s["rows"]:
            if i >= 0:
                s["s"][rows] = torch.mm(s["x"][rows].float(), s["a"][i].float().t())
    return s


def _rows_of(lens, ids):
    """(adapter, its rows): a slice where they lie together, else their numbers."""
    at, out = _offsets(lens), []
    for i in sorted(set(ids)):
        spans = [[int(at[d]), int(at[d + 1])] for d in range(len(lens)) if ids[d] == i and lens[d] > 0]
        if not spans:
            continue
        if all(a[1] == b[0] for a, b in zip(spans, spans[1:])):
            out.append((i, slice(spans[0][0], spans[-1][1])))
        else:
            out.append((i, torch.from_numpy(np.concatenate([np.arange(a, b) for a, b in spans])).cuda()))
    return out


# --- one pass ----------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if not own:
        return {"qk": _plain_qk, "qk_back": _plain_qk_back, "dropout": _plain_dropout, "adapter": _plain_adapter,
                "adapter_back": lambda s: _plain_adapter_back(s, s["s"]), "adapter_train": _plain_adapter_train}[case["op"]](s)
    nxg = _nxg()
    if case["op"] == "qk":
        return nxg.qk_norm_rope_rows(s["q"], s["k"], s["wq"], s["wk"], s["freq"], s["cu"], eps=EPS, layout=case["layout"])
    if case["op"] == "qk_back":
        return nxg.qk_norm_rope_rows_backward(s["dq_out"], s["dk_out"], s["q"], s["k"], s["wq"], s["wk"], s["freq"], s["cu"], eps=EPS,
                                              layout=case["layout"])
    if case["op"] == "dropout":
        return nxg.dropout_rows(s["x"], case["p"], case["rng"], case["offset"], residual=s["residual"])
    if case["op"] == "adapter_back":
        return nxg.adapter_rows_backward(s["dy"], s["x"], s["a"], s["b"], s["s"], s["cu"], s["ids"], s["scale"], base=s["dx_base"])
    y, low = nxg.adapter_rows(s["x"], s["a"], s["b"], s["cu"], s["ids"], s["scale"], base=s["base"])
    if case["op"] == "adapter":
        return y, low
    return (y, low) + tuple(nxg.adapter_rows_backward(s["dy"], s["x"], s["a"], s["b"], low, s["cu"], s["ids"], s["scale"],
                                                      base=s["dx_base"]))


# --- the plain forms: 32 bits, elementary operations ---------------------------------------------

def _angles(s):
    pos = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.float64)
    starts = torch.repeat_interleave(s["cu"][:-1].double(), torch.diff(s["cu"]).long())
    angle = (pos - starts)[:, None] * s["freq"][None, :]
    return torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]


def _turned(case, x, cos, sin):
    n, out = case["rot"], x.clone()
    if case["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        out[..., :n // 2] = a * cos - b * sin
        out[..., n // 2:n] = a * sin + b * cos
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        out[..., 0:n:2] = a * cos - b * sin
        out[..., 1:n:2] = a * sin + b * cos
    return out


def _plain_qk(s):
    cos, sin = _angles(s)
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x32 = x.float()
        rstd = 1.0 / torch.sqrt((x32 * x32).mean(2, keepdim=True) + EPS)
        out.append(_turned(s["case"], x32 * rstd * w.float(), cos, sin).to(x.dtype))
    return tuple(out)


def _plain_qk_back(s):
    cos, sin = _angles(s)
    dx, dw = [], []
    for dy, x, w in ((s["dq_out"], s["q"], s["wq"]), (s["dk_out"], s["k"], s["wk"])):
        u = _turned(s["case"], dy.float(), cos, -sin)
        x32 = x.float()
        rstd = 1.0 / torch.sqrt((x32 * x32).mean(2, keepdim=True) + EPS)
        h = x32 * rstd
        g = u * w.float()
        dx.append((rstd * (g - h * (g * h).mean(2, keepdim=True))).to(x.dtype))
        dw.append((u * h).sum((0, 1), dtype=torch.float64).to(w.dtype))
    return tuple(dx + dw)


def _plain_dropout(s):
    """Philox 4x32-10 (Salmon, Moraes, Dror, Shaw, 2011): the counter is (column / 8, row, offset's low and high words), the
    key the seed's two words; column c takes the 16 bits 16 (c % 2) of word (c % 8) / 2 and is dropped where they are
    below round(p 2^16)."""
    case, x = s["case"], s["x"]
    T, cols = x.shape
    low = 0xFFFFFFFF
    c0 = torch.arange((cols + 7) // 8, device="cuda").repeat(T)
    c1 = torch.arange(T, device="cuda").repeat_interleave((cols + 7) // 8)
    c2, c3 = torch.full_like(c0, case["offset"] & low), torch.full_like(c0, case["offset"] >> 32)
    k0, k1 = case["rng"] & low, case["rng"] >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57                    # modulo 2^64
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(T, -1)[:, :cols]
    least = round(case["p"] * 65536)
    y = torch.where(bits >= least, x.float() * (65536.0 / (65536 - least)), torch.zeros((), device="cuda"))
    return (y if s["residual"] is None else s["residual"].float() + y).to(x.dtype)


def _plain_adapter(s):
    x, case = s["x"], s["case"]
    y = torch.zeros(x.shape[0], case["n_out"], dtype=x.dtype, device="cuda") if s["base"] is None else s["base"].clone()
    low = torch.zeros(x.shape[0], case["rank"], device="cuda")
    if len(s["rows"]) > 4 and x.shape[0] == s["ids"].shape[0]:       # requests of one row each: all at once
        at = s["ids"].clamp(min=0).long()
        some = (s["ids"] >= 0)[:, None]
        low = torch.bmm(s["a"][at].float(), x.float()[:, :, None])[:, :, 0] * some
        d = s["scale"] * torch.bmm(s["b"][at].float(), low[:, :, None])[:, :, 0]
        return torch.where(some, y.float() + d, y.float()).to(x.dtype), low
    for i, rows in s["rows"]:
        if i >= 0:
            low[rows] = torch.mm(x[rows].float(), s["a"][i].float().t())
            y[rows] = (y[rows].float() + s["scale"] * torch.mm(low[rows], s["b"][i].float().t())).to(x.dtype)
    return y, low


def _plain_adapter_back(s, low):
    x, dy, case = s["x"], s["dy"], s["case"]
    dx = torch.zeros_like(x) if s["dx_base"] is None else s["dx_base"].clone()
    da, db = torch.zeros_like(s["a"]), torch.zeros_like(s["b"])
    for i, rows in s["rows"]:
        if i >= 0:
            dy32 = dy[rows].float()
            g = s["scale"] * torch.mm(dy32, s["b"][i].float())
            dx[rows] = (dx[rows].float() + torch.mm(g, s["a"][i].float())).to(x.dtype)
            da[i] = torch.mm(g.t(), x[rows].float()).to(da.dtype)
            db[i] = (s["scale"] * torch.mm(dy32.t(), low[rows])).to(db.dtype)
    return dx, da, db


def _plain_adapter_train(s):
    y, low = _plain_adapter(s)
    return (y, low) + _plain_adapter_back(s, low)


# --- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("qk", "qk_back"):
        return _exact_qk(case, s)
    if case["op"] == "dropout":
        keep = torch.from_numpy(_exact_kept(case)).cuda()
        y = s["x"].double() / (1.0 - round(case["p"] * 65536) / 65536) * keep
        return y if s["residual"] is None else y + s["residual"].double()
    return _exact_adapter(case, s)


def _exact_qk(case, s):
    """Each pair as a complex number times e^(i * position * frequency); the gradients by differentiation."""
    pos = np.concatenate([np.arange(n) for n in s["lens"]])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.from_numpy(pos[:, None, None] * _frequencies(case)).cuda())
    n, out, grads = case["rot"], [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s["w" + name].double()
        if case["op"] == "qk_back":
            x, w = x.requires_grad_(), w.requires_grad_()
        y = x / x.square().mean(2, keepdim=True).add(EPS).sqrt() * w
        if case["layout"] == "half":
            z = torch.complex(y[..., :n // 2], y[..., n // 2:n]) * turn
            y = torch.cat([z.real, z.imag, y[..., n:]], -1)
        else:
            z = torch.view_as_complex(y[..., :n].reshape(*y.shape[:2], n // 2, 2).contiguous()) * turn
            y = torch.cat([torch.view_as_real(z).flatten(2), y[..., n:]], -1)
        out.append(y)
        if case["op"] == "qk_back":
            grads.append(torch.autograd.grad(y, (x, w), s[f"d{name}_out"].double()))
    if case["op"] == "qk":
        return tuple(out)
    return grads[0][0], grads[1][0], grads[0][1], grads[1][1]


def _exact_kept(case):
    """[rows][cols]: is the value kept, from the generator's definition in unsigned 64-bit words, a block of rows at a time."""
    u = lambda n: np.uint64(n)                                               # noqa: E731
    cols, least = case["cols"], round(case["p"] * 65536)
    groups = np.arange((cols + 7) // 8, dtype=np.uint64)
    keep = np.empty((case["rows"], cols), np.bool_)
    step = max(1, (1 << 18) // groups.size)
    for r in range(0, case["rows"], step):
        rows = np.arange(r, min(r + step, case["rows"]), dtype=np.uint64)
        shape = (rows.size, groups.size)
        c = [np.broadcast_to(groups, shape), np.broadcast_to(rows[:, None], shape),
             np.full(shape, case["offset"] % 2 ** 32, np.uint64), np.full(shape, case["offset"] // 2 ** 32, np.uint64)]
        key = [case["rng"] % 2 ** 32, case["rng"] // 2 ** 32]
        for _ in range(10):
            a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
            c = [(b >> u(32)) ^ c[1] ^ u(key[0]), b & u(2 ** 32 - 1), (a >> u(32)) ^ c[3] ^ u(key[1]), a & u(2 ** 32 - 1)]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        drawn = np.empty(shape + (8,), np.uint16)
        for j in range(8):
            drawn[..., j] = (c[j // 2] >> u(16 * (j % 2))) & u(0xFFFF)
        keep[r:r + rows.size] = drawn.reshape(rows.size, -1)[:, :cols] >= least
    return keep


def _exact_adapter(case, s):
    """Document by document; the gradients of x and A by differentiation, B's from the forward call's s."""
    x, a, b = s["x"].double(), s["a"].double(), s["b"].double()
    T = x.shape[0]
    low = torch.zeros(T, case["rank"], dtype=torch.float64, device="cuda")
    y = torch.zeros(T, case["n_out"], dtype=torch.float64, device="cuda")
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    t = 0
    for n, i in zip(_numbers(case), _numbers(case, "ids")):
        rows, t = slice(t, t + n), t + n
        if i < 0:
            continue
        xd, ad = x[rows].requires_grad_(), a[i].clone().requires_grad_()
        ld = torch.mm(xd, ad.t())
        yd = torch.mm(ld, b[i].t()) * s["scale"]
        low[rows], y[rows] = ld.detach(), yd.detach()
        if case["op"] != "adapter":
            dy = s["dy"][rows].double()
            dx[rows], g = torch.autograd.grad(yd, (xd, ad), dy)
            da[i] += g
            db[i] += torch.mm(dy.t(), (s["s"][rows].double() if "s" in s else low[rows])) * s["scale"]
    if case["base"] and case["op"] != "adapter_back":
        y += s["base"].double()
    if case["base"] and case["op"] != "adapter":
        dx += s["dx_base"].double()
    return {"adapter": (y, low), "adapter_back": (dx, da, db), "adapter_train": (y, low, dx, da, db)}[case["op"]]
