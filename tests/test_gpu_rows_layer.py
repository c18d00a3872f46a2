"""GPU: the row operators as a layer uses them, forward and back: layer norm, a fused projection, rotary
positions on its queries and keys in place, attention, and their gradients in turn. Each step against 64
bits on its own inputs, the whole against 64-bit differentiation; captured into a graph and replayed; on
another stream; two at once."""
from __future__ import annotations

import numpy as np
import pytest

import rows_ref

pytestmark = pytest.mark.gpu

C, H, G, D = 256, 4, 2, 64
LENS = [70, 1, 130, 33]


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


class Layer:
    """One layer's path with everything that it writes allocated beforehand."""

    def __init__(self, nxg, torch, dtype, lens=LENS, seed=0):
        self.nxg, self.torch, self.lens = nxg, torch, lens
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        T = sum(lens)
        self.x, self.w, self.b = rnd(T, C).to(dtype), 1 + 0.1 * rnd(C), 0.1 * rnd(C)
        self.proj = (rnd(C, (H + 2 * G) * D) / 16).to(dtype)
        self.dout = (0.1 * rnd(T, H, D)).to(dtype)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        f, self.m = nxg.rope_frequencies(32, 10000.0, "by_parts", 2.0, 64)
        self.f = torch.from_numpy(f).cuda()

    def forward(self):
        n, t = self.nxg, self.torch
        self.y, self.mean, self.rstd = n.layer_norm_rows(self.x, self.w, self.b)
        self.plain = t.mm(self.y, self.proj).view(-1, H + 2 * G, D)
        self.qkv = self.plain.clone()
        turned = self.qkv[:, :H + G]
        n.rope_rows(turned, self.f, self.cu, mscale=self.m, out=turned)
        self.q, self.k, self.v = self.qkv[:, :H], self.qkv[:, H:H + G], self.qkv[:, H + G:]
        self.out, self.lse = n.attention_rows(self.q, self.k, self.v, self.cu, right=0)
        return self.out

    def backward(self):
        n, t = self.nxg, self.torch
        self.dqkv = t.empty_like(self.qkv)
        dq, dk, dv = self.dqkv[:, :H], self.dqkv[:, H:H + G], self.dqkv[:, H + G:]
        n.attention_rows_backward(self.dout, self.q, self.k, self.v, self.out, self.lse, self.cu, right=0, dq=dq, dk=dk, dv=dv)
        self.d_turned = self.dqkv.clone()
        turned = self.dqkv[:, :H + G]
        n.rope_rows(turned, self.f, self.cu, mscale=self.m, inverse=True, out=turned)
        flat = self.dqkv.view(-1, (H + 2 * G) * D)
        self.dy = t.mm(flat, self.proj.t().contiguous())
        self.dx, self.dw, self.db = n.layer_norm_rows_backward(self.dy, self.x, self.mean, self.rstd, self.w)
        return self.dx, self.dw, self.db

    def step(self):
        return (self.forward(),) + self.backward()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_each_step(nxg, torch, dev, dtype):
    say(f"a layer's path {dtype}, step by step")
    a = Layer(nxg, torch, getattr(torch, dtype))
    a.step()
    pos = torch.from_numpy(np.concatenate([np.arange(n) for n in LENS])).cuda()
    rows_ref.check("norm", a.y, *rows_ref.layer_norm(a.x, a.w, a.b, 1e-5)[0])
    rows_ref.check("rope", a.qkv[:, :H + G], *rows_ref.rope(a.plain[:, :H + G], a.f, pos, "half", a.m, False))
    assert torch.equal(a.qkv[:, H + G:], a.plain[:, H + G:])
    cu = a.cu.cpu().numpy()
    ref = rows_ref.attention(a.q, a.k, a.v, cu, cu, 0.125, -1, 0, a.dout)
    rows_ref.check("out", a.out, *ref["out"])
    for name, t in (("dq", a.d_turned[:, :H]), ("dk", a.d_turned[:, H:H + G]), ("dv", a.d_turned[:, H + G:])):
        rows_ref.check(name, t, *ref[name])
    rows_ref.check("rope back", a.dqkv[:, :H + G], *rows_ref.rope(a.d_turned[:, :H + G], a.f, pos, "half", a.m, True))
    for name, t, r in zip(("dx", "dw", "db"), (a.dx, a.dw, a.db), rows_ref.layer_norm_back(a.dy, a.x, a.mean, a.rstd, a.w)):
        rows_ref.check(name, t, *r)


def test_whole_against_differentiation(nxg, torch, dev):
    """The path's gradients against 64-bit differentiation of the whole. fp16: the forward path rounds 5 times
    (norm, projection, rotation, P, out), the backward path 7 (P, dS, out's share in delta, dq/dk/dv, rotation,
    product, dx), each by at most 2^-11 of its values; the softmax's slope at scores of about 1 passes an error in
    q or k on with a factor of less than 4."""
    say("a layer's path fp16 against 64-bit differentiation")
    a = Layer(nxg, torch, torch.float16)
    _, dx, dw, db = a.step()
    x, w, b = (t.double().requires_grad_() for t in (a.x, a.w, a.b))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w + b
    qkv = (y @ a.proj.double()).view(-1, H + 2 * G, D)
    pos = torch.from_numpy(np.concatenate([np.arange(n) for n in LENS])).cuda().double()
    ang = pos[:, None] * a.f[None, :]
    c, s = torch.cos(ang)[:, None] * a.m, torch.sin(ang)[:, None] * a.m
    t = qkv[:, :H + G]
    t = torch.cat([t[..., :16] * c - t[..., 16:32] * s, t[..., :16] * s + t[..., 16:32] * c, t[..., 32:]], 2)
    loss, r = 0.0, 0
    for n in LENS:
        for h in range(H):
            q, k, v = t[r:r + n, h], t[r:r + n, H + h // 2], qkv[r:r + n, H + G + h // 2]
            p = torch.softmax((q @ k.t() * 0.125).masked_fill(~rows_ref.window(n, n, -1, 0, "cuda"), -np.inf), 1)
            loss = loss + ((p @ v) * a.dout[r:r + n, h].double()).sum()
        r += n
    for name, got, ref in zip(("dx", "dw", "db"), (dx, dw, db), torch.autograd.grad(loss, (x, w, b))):
        rel = float((got.double() - ref).norm() / ref.norm())
        assert rel <= 12 * 4 * 2.0 ** -11, (name, rel)


def test_replayed_from_a_graph(nxg, torch, dev):
    """A captured step, replayed with other inputs and other documents in the same memory, eager steps between."""
    say("a layer's path captured and replayed")
    a, eager = Layer(nxg, torch, torch.bfloat16), Layer(nxg, torch, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = a.step()
    for seed, lens in ((1, LENS), (2, [234]), (3, [0, 100, 0, 134]), (4, LENS)):
        lens = lens + [0] * (len(LENS) - len(lens))
        fresh = Layer(nxg, torch, torch.bfloat16, lens, seed)
        for name in ("x", "w", "b", "proj", "dout", "cu"):
            getattr(a, name).copy_(getattr(fresh, name))
        graph.replay()
        torch.cuda.synchronize()
        want = fresh.step()
        eager.step()
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(outs, want)):
            assert torch.equal(x, y), (seed, i)


def test_on_another_stream_and_two_at_once(nxg, torch, dev):
    say("a layer's path on other streams")
    a = [Layer(nxg, torch, torch.bfloat16, [500, 90], s) for s in (1, 2)]
    want = [[t.clone() for t in l.step()] for l in a]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in a]
    got = [None, None]
    for _ in range(5):
        for i, (l, s) in enumerate(zip(a, streams)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = l.step()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    # the stream argument, with host offsets made on the current stream
    l, s = a[0], streams[0]
    out, lse = nxg.attention_rows(l.q, l.k, l.v, [0, 500, 590], right=0, stream=s)
    grads = nxg.attention_rows_backward(l.dout, l.q, l.k, l.v, out, lse, [0, 500, 590], right=0, stream=s)
    y = nxg.layer_norm_rows(l.x, l.w, l.b, stream=s)[0]
    s.synchronize()
    assert torch.equal(out, l.out) and torch.equal(grads[0], l.d_turned[:, :H]) and torch.equal(y, l.y)


def test_caller_workspaces(nxg, torch, dev):
    """A workspace of the caller's is used within its size and no further; one that is too small is refused."""
    say("workspaces of the caller")
    a = Layer(nxg, torch, torch.float16)
    a.step()
    args = (a.q, a.k, a.v, a.cu)
    n = nxg.attention_rows_backward_workspace_bytes(*args, right=0)
    ws = torch.full((n + 64,), 7, dtype=torch.uint8, device="cuda")
    grads = nxg.attention_rows_backward(a.dout, *args[:3], a.out, a.lse, a.cu, right=0, workspace=ws[:n])
    assert torch.equal(grads[0], a.d_turned[:, :H]) and (ws[n:] == 7).all()
    with pytest.raises(ValueError, match="workspace"):
        nxg.attention_rows_backward(a.dout, *args[:3], a.out, a.lse, a.cu, right=0, workspace=ws[:n - 16])
    m = nxg.layer_norm_rows_workspace_bytes(*a.x.shape)
    ws = torch.full((m + 64,), 7, dtype=torch.uint8, device="cuda")
    dx, dw, db = nxg.layer_norm_rows_backward(a.dy, a.x, a.mean, a.rstd, a.w, workspace=ws[:m])
    assert torch.equal(dw, a.dw) and torch.equal(db, a.db) and (ws[m:] == 7).all()
    with pytest.raises(ValueError, match="workspace"):
        nxg.layer_norm_rows_backward(a.dy, a.x, a.mean, a.rstd, a.w, workspace=ws[:m - 16])
    with pytest.raises(ValueError):
        nxg.attention_rows(*args, lse=torch.empty(1, device="cuda"))
    with pytest.raises(ValueError):
        nxg.attention_rows(a.q, a.k, a.v[:-1], a.cu)
    with pytest.raises(ValueError):
        nxg.attention_rows(a.q, a.k, a.v, a.cu, a.cu[:-1])
    with pytest.raises(ValueError):
        nxg.rope_rows(a.q, a.f, a.cu, positions=a.cu)
