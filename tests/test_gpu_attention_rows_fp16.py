"""GPU: attention_rows and its gradients in fp16, whose range P and dS leave: each row's results are as exact as its own values
allow, whatever other documents, or other tokens of its document, hold (and bf16, which has no such limits)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import rows_ref

pytestmark = pytest.mark.gpu
F32 = rows_ref.F32


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.fixture(scope="module")
def dev(torch, nxg):
    nxg.init()
    return torch.device("cuda:0")


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def make(torch, dtype, T, H, G, D, seed, grad=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, do = (torch.randn(T, n, D, device="cuda", generator=g) for n in (H, G, G, H))
    return q.to(dtype), k.to(dtype), v.to(dtype), (grad * do).to(dtype)


def run(nxg, q, k, v, do, cu, left, right):
    out, lse = nxg.attention_rows(q, k, v, cu, left=left, right=right)
    return (out, lse) + tuple(nxg.attention_rows_backward(do, q, k, v, out, lse, cu, left=left, right=right))


def check_documents(torch, got, q, k, v, do, lens, left, right, which):
    """The documents `which` against 64 bits, with bounds from each one's own values: as a call of that document alone."""
    cu = offsets(lens)
    for d in which:
        s = slice(int(cu[d]), int(cu[d + 1]))
        ref = rows_ref.attention(q[s], k[s], v[s], [0, lens[d]], [0, lens[d]], 1 / math.sqrt(q.shape[2]), left, right, do[s])
        for name, t in zip(("out", "lse", "dq", "dk", "dv"), got):
            rows_ref.check(f"document {d}: {name}", t[s], *ref[name])


TYPES = ["float16", "bfloat16"]


@pytest.mark.parametrize("dtype,size", [("float16", (100.0, 30.0)), ("float16", (8000.0, 1000.0)), ("bfloat16", (8000.0, 1000.0))], ids=str)
@pytest.mark.parametrize("lens", [[200, 70, 33], [1000, 300, 64]], ids=str)
@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (2, 1, 128)])
def test_another_documents_sizes(nxg, torch, dev, H, G, D, lens, dtype, size):
    """dout and v of one document up to 2^23 and 2^10 times another's."""
    print(f"attention_rows {dtype} H={H} D={D} {lens}: a document of {size}", flush=True)
    q, k, v, do = make(torch, getattr(torch, dtype), sum(lens), H, G, D, 1)
    s = slice(lens[0], lens[0] + lens[1])
    do[s] = (do[s].float() * (size[0] / 1e-3)).clamp(-60000, 60000).to(do.dtype)
    v[s] *= size[1]
    got = run(nxg, q, k, v, do, offsets(lens), -1, 0)
    check_documents(torch, got, q, k, v, do, lens, -1, 0, [0, 2])
    assert all(bool(torch.isfinite(t[:lens[0]]).all()) for t in got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", ["dout", "v", "both"])
@pytest.mark.parametrize("value", [-math.inf, math.nan])
def test_another_documents_infinities(nxg, torch, dev, value, bad, dtype):
    """One value of another document that is not finite."""
    print(f"attention_rows {dtype} {value} in another document's {bad}", flush=True)
    lens = [500, 40, 90]
    q, k, v, do = make(torch, getattr(torch, dtype), sum(lens), 4, 2, 64, 2, 1e-4)
    if bad != "v":
        do[510, 1, 3] = value
    if bad != "dout":
        v[511, 0, 7] = value
    for left, right in ((-1, 0), (-1, -1), (20, 20)):
        got = run(nxg, q, k, v, do, offsets(lens), left, right)
        check_documents(torch, got, q, k, v, do, lens, left, right, [0, 2])


def gradients(torch, q, k, v, do, left, right, u, out_bound):
    """One document's {"dq", "dk", "dv"}: (value, bound) in 64 bits, for finite inputs. dS is rounded once to the type, off by u of
    it, or, below the type's normal numbers, by 2^-34 of the largest dS of its own row (dq: of the query, dk: of the key): a row
    of dS is carried so that its largest is at least 2^9, in steps of 2^-24 at least. P is carried as 2^15 P. The rest are fp32
    sums and exponentials as in rows_ref, and delta's share of the output's error."""
    n, H, D = q.shape
    G, R, scale = k.shape[1], q.shape[1] // k.shape[1], 1 / math.sqrt(D)
    seen = rows_ref.window(n, n, left, right, q.device)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    res = {x: [torch.zeros(n, w, D, dtype=torch.float64, device=q.device) for _ in range(2)] for x, w in (("dq", H), ("dk", G), ("dv", G))}
    least = rows_ref.least_step(q.dtype)
    for g in range(G):
        K, V = k[:, g].double(), v[:, g].double()
        col = []
        for h in range(g * R, (g + 1) * R):
            Q, dO = q[:, h].double(), do[:, h].double()
            S = torch.where(seen, (Q @ K.t()) * scale, -math.inf)
            es = torch.where(seen, (D + 8) * F32 * scale * (Q.abs() @ K.abs().t()), zero).amax(1, keepdim=True)
            ep = 2 * es + 8 * F32 * (torch.where(seen, S.abs(), zero).amax(1, keepdim=True) + 1) + n * F32
            P = torch.where(seen, torch.exp(S - torch.logsumexp(S, 1, keepdim=True)), zero)
            O = P @ V
            dP = torch.where(seen, dO @ V.t(), zero)
            delta = (dO * O).sum(1, keepdim=True)
            e_delta = (dO.abs() * out_bound[:, h]).sum(1, keepdim=True) + (D + 4) * F32 * (dO.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (dP - delta)
            e_ds = P * (e_delta + (D + 4) * F32 * torch.where(seen, dO.abs() @ V.abs().t(), zero)) * (1 + 4 * ep) \
                + dS.abs() * (u * 1.01 + 4 * ep + (n + 8) * F32) + P * delta.abs() * 4 * F32 + seen * 2.0 ** -85
            steps = lambda axis: seen * ((dS.abs() + e_ds).amax(axis, keepdim=True) * 2.0 ** -34)  # noqa: E731
            dQ = dS @ K * scale
            res["dq"][0][:, h] = dQ
            res["dq"][1][:, h] = ((e_ds + steps(1)) @ K.abs()) * scale + 1.01 * u * dQ.abs() + least
            col.append((dS, e_ds, Q, P, ep, dO))
        top = torch.stack([(a.abs() + b).amax(0) for a, b, *_ in col]).amax(0) * 2.0 ** -34       # of a key, over its heads
        for dS, e_ds, Q, P, ep, dO in col:
            res["dk"][0][:, g] += dS.t() @ Q * scale
            res["dk"][1][:, g] += (e_ds + seen * top[None, :] + n * F32 * dS.abs()).t() @ Q.abs() * scale
            res["dv"][0][:, g] += P.t() @ dO
            res["dv"][1][:, g] += (P * (1.01 * u + 4 * ep + (n + 8) * F32) + seen * 2.0 ** -39).t() @ dO.abs()
        for x in ("dk", "dv"):
            res[x][1][:, g] = 1.01 * res[x][1][:, g] + 1.01 * u * res[x][0][:, g].abs() + least
    return res


@pytest.mark.parametrize("H,G,D,n,dtype", [(4, 2, 64, 300, "float16"), (2, 1, 64, 1500, "float16"), (2, 2, 128, 700, "float16"), (6, 2, 40, 260, "bfloat16")])
@pytest.mark.parametrize("left,right", [(-1, 0), (30, 30), (-1, -1)])
@pytest.mark.parametrize("what", ["dout", "v", "both"])
def test_tokens_of_other_sizes(nxg, torch, dev, what, left, right, H, G, D, n, dtype):
    """Tokens of one document whose dout and v differ by up to 2^20, rising and falling along it and from token to token."""
    print(f"attention_rows {dtype} H={H} D={D} {n} tokens, window={left},{right}: {what} of sizes 2^-10 to 2^10", flush=True)
    dt = getattr(torch, dtype)
    q, k, v, do = make(torch, dt, n, H, G, D, 3, 1.0)
    g = torch.Generator(device="cuda").manual_seed(7)
    waves = torch.cos(torch.arange(n, device="cuda") * (2 * math.pi / n * 2.5)) * 10
    jumps = torch.randint(-10, 11, (n,), device="cuda", generator=g)
    for sizes in (waves.round(), jumps.float()):
        f = torch.exp2(sizes)[:, None, None]
        d2 = (do.float() * f).to(dt) if what != "v" else do
        v2 = (v.float() * f.flip(0)).to(dt) if what != "dout" else v
        out, lse, dq, dk, dv = run(nxg, q, k, v2, d2, offsets([n]), left, right)
        ref = rows_ref.attention(q, k, v2, [0, n], [0, n], 1 / math.sqrt(D), left, right)
        rows_ref.check("out", out, *ref["out"])
        want = gradients(torch, q, k, v2, d2, left, right, rows_ref.half_step(dt), ref["out"][1])
        for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
            # a value past the type's largest number rounds to infinity
            value, bound = want[name]
            past = (value.abs() + bound >= torch.finfo(dt).max) & torch.isinf(t) & (torch.sign(t) == torch.sign(value))
            rows_ref.check(name, torch.where(past, torch.zeros_like(t), t), torch.where(past, torch.zeros_like(value), value), bound)


def test_a_document_alone_and_in_a_batch(nxg, torch, dev):
    """The same bits with any other document beside it, where both calls take the documents whole."""
    lens = [512] * 12
    q, k, v, do = make(torch, torch.float16, sum(lens), 8, 8, 64, 4)
    cu = offsets(lens)
    plain = run(nxg, q, k, v, do, cu, -1, 0)
    s = slice(512, 1024)
    do[s] *= 1000
    v[s] *= 1000
    do[s][7, 3, 5] = math.inf
    print("attention_rows fp16: twelve documents, one of them changed", flush=True)
    for a, b in zip(plain, run(nxg, q, k, v, do, cu, -1, 0)):
        assert torch.equal(a[:512], b[:512]) and torch.equal(a[1024:], b[1024:])


def forward(torch, q, k, v, n, m, left, right, u, step):
    """One document's (out, bound), as rows_ref's, where a carried weight is off by u of it, or by `step` of the largest."""
    H, G, D = q.shape[1], k.shape[1], q.shape[2]
    value, bound = (torch.zeros(n, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    seen = rows_ref.window(n, m, left, right, q.device)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    for h in range(H):
        Q, K, V = q[:, h].double(), k[:, h // (H // G)].double(), v[:, h // (H // G)].double()
        S = torch.where(seen, (Q @ K.t()) / math.sqrt(D), -math.inf)
        es = torch.where(seen, (D + 8) * F32 / math.sqrt(D) * (Q.abs() @ K.abs().t()), zero).amax(1, keepdim=True)
        # a sum takes 16 keys at once, with 4 roundings at most
        ep = 2 * es + 8 * F32 * (torch.where(seen, S.abs(), zero).amax(1, keepdim=True) + 1) + (m / 4 + 64) * F32
        P = torch.exp(S - torch.logsumexp(S, 1, keepdim=True))
        value[:, h] = P @ V
        bound[:, h] = (1.01 * u + 2 * ep) * (P @ V.abs()) + u * value[:, h].abs() + step * (seen.double() @ V.abs()) + rows_ref.least_step(q.dtype)
    return value, bound


@pytest.mark.parametrize("n,m,H,G,D,dtype", [(1, 65536, 4, 2, 64, "float16"), (3, 30000, 2, 1, 96, "float16"), (700, 16384, 4, 4, 64, "float16"),
                                             (700, 16384, 4, 4, 96, "float16"), (700, 16384, 4, 4, 64, "bfloat16"), (1, 1 << 20, 1, 1, 64, "float16")])
@pytest.mark.parametrize("above", [14.0, 17.3])
@pytest.mark.parametrize("at", [0, 0.4])
def test_many_small_weights_beside_a_large_one(nxg, torch, dev, at, above, n, m, H, G, D, dtype):
    """One key so far above all others (in nats) that each of them alone would be lost, but not their sum. A weight is carried with
    the largest at 2^10 at least when it came, so that fp16's half step of 2^-25 is 2^-35 of it."""
    print(f"attention_rows {dtype} {n} queries over {m} keys, one of them {above} above", flush=True)
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(m)
    q = torch.zeros(n, H, D, device="cuda")
    q[:, :, 0] = 1
    k = torch.zeros(m, G, D, device="cuda")
    k[int(at * (m - 1)), :, 0] = above * math.sqrt(D)
    v = 1 + 0.25 * torch.randn(m, G, D, device="cuda", generator=g)
    v[int(at * (m - 1))] = -0.01
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    out, _ = nxg.attention_rows(q, k, v, [0, n], [0, m])
    step = 2.0 ** -35 if dt == torch.float16 else 0.0
    rows_ref.check("out", out, *forward(torch, q, k, v, n, m, -1, -1, rows_ref.half_step(dt), step))


@pytest.mark.parametrize("size", [0.5, 3.0, 10.0, 60.0])
@pytest.mark.parametrize("n,m,H,G,left,right", [(1, 20000, 4, 2, -1, -1), (1500, 1500, 4, 2, -1, 0), (900, 900, 8, 8, 100, 100), (40, 3000, 2, 2, -1, 0)])
def test_scores_of_all_sizes(nxg, torch, dev, n, m, H, G, left, right, size):
    """Scores spread by `size`, rising along the keys too, so that the reference is raised now and then, or in every tile."""
    print(f"attention_rows fp16 {n} over {m} keys, scores of +-{size}", flush=True)
    D, dt = 64, torch.float16
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k, v = (torch.randn(x, y, D, device="cuda", generator=g) for x, y in ((n, H), (m, G), (m, G)))
    for ramp in (torch.ones(m, device="cuda"), torch.linspace(0.02, 1, m, device="cuda")):
        a, b, c = (q * size).to(dt), (k * ramp[:, None, None]).to(dt), v.to(dt)
        out, lse = nxg.attention_rows(a, b, c, [0, n], [0, m], left=left, right=right)
        rows_ref.check("out", out, *forward(torch, a, b, c, n, m, left, right, rows_ref.half_step(dt), 2.0 ** -35))
        rows_ref.check("lse", lse, *rows_ref.attention(a, b, c, [0, n], [0, m], 1 / math.sqrt(D), left, right)["lse"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("left,right,D", [(-1, 0, 64), (7, 7, 128), (40, -1, 64)])
def test_infinities_inside_a_document(nxg, torch, dev, left, right, D, bad, dtype):
    """Infinities of either sign in some tokens of one input: whatever does not depend on them (what stays finite in 64 bits with
    NaN in their place) is as without. What does is not defined: a softmax of infinite scores, sums of both signs."""
    print(f"attention_rows_backward {dtype} D={D} window={left},{right}: infinities in {bad}", flush=True)
    dt = getattr(torch, dtype)
    lens = [150, 75]
    tensors = dict(zip(("q", "k", "v", "dout"), make(torch, dt, sum(lens), 4, 2, D, 5, 0.1)))
    for i, t in enumerate((100, 149, 160)):
        tensors[bad][t, i % 2, 3 * i] = math.inf if i % 2 else -math.inf
    q, k, v, do = tensors.values()
    got = run(nxg, q, k, v, do, offsets(lens), left, right)
    q, k, v, do = (torch.where(torch.isinf(t), torch.full_like(t, math.nan), t) for t in (q, k, v, do))
    ref = rows_ref.attention(q, k, v, offsets(lens), offsets(lens), 1 / math.sqrt(D), left, right, do)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), got):
        value, bound = ref[name]
        exact, zero = torch.isfinite(value), torch.zeros((), dtype=torch.float64, device=t.device)
        assert bool(exact.any())
        rows_ref.check(name, torch.where(exact, t.double(), zero), torch.where(exact, value, zero), torch.where(exact, bound, zero))
