"""GPU: the row operators of adapter fine-tuning as a layer uses them, forward and back: a frozen int8 projection with adapters
on its fp32 rows, head norms with rotation in place, attention, an output projection with adapters, dropout with the residual, and
their gradients in turn. Each step against 64 bits on its own inputs, the whole against 64-bit differentiation; captured into a graph
and replayed; on other streams; two at once; with the caller's workspaces."""
from __future__ import annotations

import numpy as np
import pytest

import adapter_ref
import rows_ref

pytestmark = pytest.mark.gpu

C, H, G, D, R, N = 256, 4, 2, 64, 16, 3
E = (H + 2 * G) * D
LENS, IDS = [70, 1, 130, 33], [1, 0, -1, 1]
SCALE, P, SEED = 2.0, 0.1, 1234567890123


def say(msg):
    print(msg, flush=True)


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.fixture(scope="module")
def dev(torch, nxg):
    nxg.init()
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def frozen(nxg, dev):
    """The int8 weight of queries, keys and values."""
    rows = (0.06 * np.random.default_rng(0).standard_normal((E, C))).astype(np.float32)
    return nxg.DeviceWeight(nxg.expand_weight(8, nxg.quantize_weight(8, rows), C, E))


INPUTS = ("x", "x32", "a1", "b1", "a2", "b2", "wq", "wk", "wo", "dh", "cu", "ids", "step")


class Layer:

    def __init__(self, nxg, torch, frozen, dtype, lens=LENS, ids=IDS, seed=0):
        self.nxg, self.torch, self.frozen, self.lens = nxg, torch, frozen, lens
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        T = sum(lens)
        self.x = rnd(T, C).to(dtype)
        self.x32 = self.x.float()
        self.a1, self.b1 = (rnd(N, R, C) / 16).to(dtype), (rnd(N, E, R) / 8).to(dtype)
        self.a2, self.b2 = (rnd(N, R, H * D) / 16).to(dtype), (rnd(N, C, R) / 8).to(dtype)
        self.wq, self.wk = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
        self.wo = (rnd(H * D, C) / 16).to(dtype)
        self.dh = (0.1 * rnd(T, C)).to(dtype)
        self.cu, self.ids = ints(np.concatenate([[0], np.cumsum(lens)])), ints(ids)
        self.step = torch.full((1,), seed, dtype=torch.int64, device="cuda")
        self.f = torch.from_numpy(nxg.rope_frequencies(32, 10000.0)[0]).cuda()

    def forward(self):
        n, t = self.nxg, self.torch
        self.frozen_rows = n.linear_i8(self.frozen, n.quantize_rows(self.x32))
        rows = self.frozen_rows.clone()
        self.rows, self.s1 = n.adapter_rows(self.x32, self.a1, self.b1, self.cu, self.ids, SCALE, base=rows, out=rows)
        self.plain = self.rows.to(self.x.dtype).view(-1, H + 2 * G, D)
        self.qkv = self.plain.clone()
        self.q, self.k, self.v = self.qkv[:, :H], self.qkv[:, H:H + G], self.qkv[:, H + G:]
        n.qk_norm_rope_rows(self.q, self.k, self.wq, self.wk, self.f, self.cu, q_out=self.q, k_out=self.k)
        self.out, self.lse = n.attention_rows(self.q, self.k, self.v, self.cu, right=0)
        self.flat = self.out.view(-1, H * D)
        self.proj = t.mm(self.flat, self.wo)
        self.y, self.s2 = n.adapter_rows(self.flat, self.a2, self.b2, self.cu, self.ids, SCALE, base=self.proj)
        return n.dropout_rows(self.y, P, SEED, 5, step=self.step, residual=self.x)

    def backward(self):
        n, t = self.nxg, self.torch
        self.dy = n.dropout_rows(self.dh, P, SEED, 5, step=self.step)
        self.dflat_base = t.mm(self.dy, self.wo.t().contiguous())
        self.dflat, da2, db2 = n.adapter_rows_backward(self.dy, self.flat, self.a2, self.b2, self.s2, self.cu, self.ids, SCALE,
                                                       base=self.dflat_base)
        self.dqkv = t.empty_like(self.qkv)
        dq, dk, dv = self.dqkv[:, :H], self.dqkv[:, H:H + G], self.dqkv[:, H + G:]
        n.attention_rows_backward(self.dflat.view(-1, H, D), self.q, self.k, self.v, self.out, self.lse, self.cu, right=0,
                                  dq=dq, dk=dk, dv=dv)
        self.d_turned = self.dqkv.clone()
        _, _, dwq, dwk = n.qk_norm_rope_rows_backward(dq, dk, self.plain[:, :H], self.plain[:, H:H + G], self.wq, self.wk, self.f, self.cu,
                                                      dq=dq, dk=dk)
        self.d32 = self.dqkv.view(-1, E).float()
        # the frozen projection passes nothing on: dx is the adapters' and the residual's
        self.dh32 = self.dh.float()
        dx, da1, db1 = n.adapter_rows_backward(self.d32, self.x32, self.a1, self.b1, self.s1, self.cu, self.ids, SCALE, base=self.dh32)
        self.grads = dict(dx=dx, da1=da1, db1=db1, da2=da2, db2=db2, dwq=dwq, dwk=dwk)
        return tuple(self.grads.values())

    def both(self):
        return (self.forward(),) + self.backward()

    def positions(self):
        return self.torch.from_numpy(np.concatenate([np.arange(n) for n in self.lens])).cuda()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_each_step(nxg, torch, dev, frozen, dtype):
    say(f"an adapted layer {dtype}, step by step")
    a = Layer(nxg, torch, frozen, getattr(torch, dtype))
    h = a.both()[0]
    check, pos, cu = rows_ref.check, a.positions(), a.cu.cpu().numpy()
    turn = (a.f, pos, "half", 1.0)

    (y, by), (s, bs) = adapter_ref.adapter(a.x32, a.a1, a.b1, cu, IDS, SCALE, a.frozen_rows)
    check("rows", a.rows, y, by)
    check("s1", a.s1, s, bs)
    check("q", a.q, *adapter_ref.qk_norm_rope(a.plain[:, :H], a.wq, *turn, 1e-6))
    check("k", a.k, *adapter_ref.qk_norm_rope(a.plain[:, H:H + G], a.wk, *turn, 1e-6))
    assert torch.equal(a.v, a.plain[:, H + G:])
    ref = rows_ref.attention(a.q, a.k, a.v, cu, cu, 0.125, -1, 0, a.dflat.view(-1, H, D))
    check("out", a.out, *ref["out"])
    (y, by), (s, bs) = adapter_ref.adapter(a.flat, a.a2, a.b2, cu, IDS, SCALE, a.proj)
    check("y", a.y, y, by)
    check("s2", a.s2, s, bs)
    check("h", h, *adapter_ref.dropout(a.y, a.x, P, SEED, 5))

    g = a.grads
    check("dy", a.dy, *adapter_ref.dropout(a.dh, None, P, SEED, 5))
    ref2 = adapter_ref.adapter_back(a.dy, a.flat, a.a2, a.b2, a.s2, cu, IDS, SCALE, a.dflat_base)
    for name, t, r in zip(("dflat", "da2", "db2"), (a.dflat, g["da2"], g["db2"]), ref2):
        check(name, t, *r)
    for name, t in (("dq", a.d_turned[:, :H]), ("dk", a.d_turned[:, H:H + G]), ("dv", a.d_turned[:, H + G:])):
        check(name, t, *ref[name])
    for name, w, heads in (("q", a.wq, slice(0, H)), ("k", a.wk, slice(H, H + G))):
        dx, dw = adapter_ref.qk_norm_rope_back(a.d_turned[:, heads], a.plain[:, heads], w, *turn, 1e-6)
        check("d" + name, a.dqkv[:, heads], *dx)
        check("dw" + name, g["dw" + name], *dw)
    ref1 = adapter_ref.adapter_back(a.d32, a.x32, a.a1, a.b1, a.s1, cu, IDS, SCALE, a.dh32)
    for name, r in zip(("dx", "da1", "db1"), ref1):
        check(name, g[name], *r)
    assert not g["da1"][2].any() and not g["db2"][2].any()


def test_whole_against_differentiation(nxg, torch, dev, frozen):
    """fp16: the forward path rounds 6 times (the rows' type, norm and rotation, P, out, projection, y), the backward path 8 (dy, its
    product, dflat, P and dS, out's share in delta, dq/dk/dv, through the norm, a gradient's own), each by at most 2^-11 of its values;
    the softmax's slope at scores of about 1 passes an error in q or k on with a factor of less than 4."""
    say("an adapted layer fp16 against 64-bit differentiation")
    a = Layer(nxg, torch, frozen, torch.float16)
    a.both()
    x, a1, b1, a2, b2, wq, wk = leaves = [t.double().requires_grad_() for t in (a.x, a.a1, a.b1, a.a2, a.b2, a.wq, a.wk)]

    def adapted(rows, base, ta, tb):
        out, r = [], 0
        for n, i in zip(LENS, IDS):
            out.append(base[r:r + n] if i < 0 else base[r:r + n] + SCALE * (rows[r:r + n] @ ta[i].t()) @ tb[i].t())
            r += n
        return torch.cat(out)

    qkv = adapted(x, a.frozen_rows.double(), a1, b1).view(-1, H + 2 * G, D)
    ang = a.positions().double()[:, None] * a.f[None, :]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def turned(t, w):
        t = t * (t.square().mean(2, keepdim=True) + 1e-6) ** -0.5 * w
        return torch.cat([t[..., :16] * c - t[..., 16:32] * s, t[..., :16] * s + t[..., 16:32] * c, t[..., 32:]], 2)

    q, k, v = turned(qkv[:, :H], wq), turned(qkv[:, H:H + G], wk), qkv[:, H + G:]
    out, r = [], 0
    for n in LENS:
        seen = rows_ref.window(n, n, -1, 0, "cuda")
        heads = [torch.softmax((q[r:r + n, h] @ k[r:r + n, h // 2].t() * 0.125).masked_fill(~seen, -np.inf), 1) @ v[r:r + n, h // 2]
                 for h in range(H)]
        out.append(torch.stack(heads, 1).reshape(n, H * D))
        r += n
    flat = torch.cat(out)
    y = adapted(flat, flat @ a.wo.double(), a2, b2)
    keep = torch.from_numpy(adapter_ref.kept(*y.shape, P, SEED, 5)).cuda()
    h = torch.where(keep, y * (65536 / (65536 - round(P * 65536))), 0.0) + x
    for name, ref in zip(("dx", "da1", "db1", "da2", "db2", "dwq", "dwk"), torch.autograd.grad((h * a.dh.double()).sum(), leaves)):
        rel = float((a.grads[name].double() - ref).norm() / ref.norm())
        say(f"{name} {rel:.2e}")
        assert rel <= 14 * 4 * 2.0 ** -11, (name, rel)


def test_replayed_from_a_graph(nxg, torch, dev, frozen):
    """A captured step, replayed with other inputs, documents, adapters and dropout steps in the same memory, eager steps between."""
    say("an adapted layer captured and replayed")
    a, eager = (Layer(nxg, torch, frozen, torch.bfloat16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = a.both()
    for seed, lens, ids in ((1, LENS, IDS), (2, [234], [2]), (3, [0, 100, 0, 134], [0, 0, 0, 0]), (4, LENS, [-1, 7, 2, 2]), (0, LENS, IDS)):
        lens, ids = lens + [0] * (len(LENS) - len(lens)), ids + [0] * (len(LENS) - len(ids))
        fresh = Layer(nxg, torch, frozen, torch.bfloat16, lens, ids, seed)
        for name in INPUTS:
            getattr(a, name).copy_(getattr(fresh, name))
        graph.replay()
        torch.cuda.synchronize()
        want = fresh.both()
        eager.both()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(outs, want)):
            assert torch.equal(p, q), (seed, i)


@pytest.mark.parametrize("n", [3, 64])
def test_single_tokens_replayed(nxg, torch, dev, n):
    """Serving: 50 requests of a token each, captured once, replayed with other adapters and with requests that end; together
    (fewer adapters than requests) or one by one."""
    say(f"single tokens of {n} adapters captured and replayed")
    g = torch.Generator(device="cuda").manual_seed(7)
    x, base = (torch.randn(50, c, device="cuda", generator=g) for c in (C, E))
    a, b = torch.randn(n, R, C, device="cuda", generator=g).bfloat16() / 16, torch.randn(n, E, R, device="cuda", generator=g).bfloat16() / 8
    cu, ids = torch.arange(51, dtype=torch.int32, device="cuda"), torch.zeros(50, dtype=torch.int32, device="cuda")
    out, s = torch.empty_like(base), torch.empty(50, R, device="cuda")
    nxg.adapter_rows(x, a, b, cu, ids, SCALE, base=base, out=out, s=s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nxg.adapter_rows(x, a, b, cu, ids, SCALE, base=base, out=out, s=s)
    for i in range(4):
        now = [(i * 5 + d * (i + 1)) % (n + 1) - 1 for d in range(50)]
        ends = np.minimum(np.arange(51), 50 - 9 * i)
        ids.copy_(torch.tensor(now, dtype=torch.int32))
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        T = int(ends[-1])
        (y, by), _ = adapter_ref.adapter(x, a, b, ends, now, SCALE, base)
        rows_ref.check("y", out[:T], y[:T], by[:T])
        assert (out[T:] == 7.0).all()
        again, _ = nxg.adapter_rows(x, a, b, cu, now, SCALE, base=base)
        assert torch.equal(again[:T], out[:T])


def test_on_other_streams_and_two_at_once(nxg, torch, dev, frozen):
    say("an adapted layer on other streams")
    a = [Layer(nxg, torch, frozen, torch.bfloat16, [500, 90], [1, 1], s) for s in (1, 2)]
    want = [[t.clone() for t in l.both()] for l in a]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in a]
    got = [None, None]
    for _ in range(5):
        for i, (l, s) in enumerate(zip(a, streams)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = l.both()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    # the stream argument, with host offsets and ids made on the current stream
    l, s, cu, ids = a[0], streams[0], [0, 500, 590], [1, 1]
    y, s2 = nxg.adapter_rows(l.flat, l.a2, l.b2, cu, ids, SCALE, base=l.proj, stream=s)
    grads = nxg.adapter_rows_backward(l.dy, l.flat, l.a2, l.b2, l.s2, cu, ids, SCALE, base=l.dflat_base, stream=s)
    q, k = l.plain[:, :H], l.plain[:, H:H + G]
    qn, kn = nxg.qk_norm_rope_rows(q, k, l.wq, l.wk, l.f, cu, stream=s)
    dqk = nxg.qk_norm_rope_rows_backward(l.d_turned[:, :H], l.d_turned[:, H:H + G], q, k, l.wq, l.wk, l.f, cu, stream=s)
    dy = nxg.dropout_rows(l.dh, P, SEED, 5, step=l.step, stream=s)
    s.synchronize()
    assert torch.equal(y, l.y) and torch.equal(s2, l.s2) and torch.equal(dy, l.dy)
    assert torch.equal(grads[0], l.dflat) and torch.equal(grads[1], l.grads["da2"]) and torch.equal(grads[2], l.grads["db2"])
    assert torch.equal(qn, l.q) and torch.equal(kn, l.k) and torch.equal(dqk[0], l.dqkv[:, :H])
    assert torch.equal(dqk[2], l.grads["dwq"]) and torch.equal(dqk[3], l.grads["dwk"])


def test_caller_workspaces(nxg, torch, dev, frozen):
    """A workspace of the caller's is used within its size and no further; one that is too small is refused."""
    say("workspaces of the caller")
    a = Layer(nxg, torch, frozen, torch.float16)
    a.both()
    args = (a.flat, a.a2, a.b2)
    n = nxg.adapter_rows_backward_workspace_bytes(*args, a.cu, a.ids)
    back = lambda ws: nxg.adapter_rows_backward(a.dy, *args, a.s2, a.cu, a.ids, SCALE, base=a.dflat_base, workspace=ws)  # noqa: E731
    ws = torch.full((n + 64,), 7, dtype=torch.uint8, device="cuda")
    grads = back(ws[:n])
    assert torch.equal(grads[0], a.dflat) and torch.equal(grads[1], a.grads["da2"]) and torch.equal(grads[2], a.grads["db2"])
    assert (ws[n:] == 7).all()
    with pytest.raises(ValueError, match="workspace"):
        back(ws[:n - 16])
    m = nxg.qk_norm_rope_rows_workspace_bytes(D)
    ws = torch.full((m + 64,), 7, dtype=torch.uint8, device="cuda")
    back = lambda ws: nxg.qk_norm_rope_rows_backward(a.d_turned[:, :H], a.d_turned[:, H:H + G], a.plain[:, :H], a.plain[:, H:H + G],  # noqa: E731
                                                     a.wq, a.wk, a.f, a.cu, workspace=ws)
    grads = back(ws[:m])
    assert torch.equal(grads[2], a.grads["dwq"]) and torch.equal(grads[3], a.grads["dwk"]) and (ws[m:] == 7).all()
    with pytest.raises(ValueError, match="workspace"):
        back(ws[:m - 16])
    # other refusals of what the functions are given
    for bad in (dict(ids=[0, 1]), dict(ids=[0.5, 1, 2, 3]), dict(cu_offsets=a.cu[:1]), dict(s=torch.empty(3, R, device="cuda")),
                dict(out=a.y[:-1]), dict(base=a.x32), dict(scale=float("inf")), dict(a=a.a2.float()), dict(b=a.b2[:, :-1])):
        kw = dict(x=a.flat, a=a.a2, b=a.b2, cu_offsets=a.cu, ids=a.ids)
        kw.update(bad)
        with pytest.raises(ValueError):
            nxg.adapter_rows(**kw)
    for bad in (dict(k=None), dict(wk=None), dict(wq=a.wq.half()), dict(k=a.k[:-1]), dict(positions=a.cu), dict(cu_offsets=None),
                dict(layout="thirds"), dict(q_out=a.k), dict(eps=float("nan"))):
        kw = dict(q=a.q, k=a.k, wq=a.wq, wk=a.wk, freq=a.f, cu_offsets=a.cu)
        kw.update(bad)
        with pytest.raises(ValueError):
            nxg.qk_norm_rope_rows(**kw)
    for bad in (dict(p=1.0), dict(p=-0.1), dict(seed=-1), dict(offset=1 << 64), dict(residual=a.x32), dict(step=a.cu), dict(out=a.x[:1])):
        kw = dict(x=a.x, p=0.5, seed=1)
        kw.update(bad)
        with pytest.raises(ValueError):
            nxg.dropout_rows(**kw)
