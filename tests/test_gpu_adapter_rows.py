"""GPU: adapter_rows and adapter_rows_backward against 64 bits (adapter_ref.py, with the bounds of their roundings)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import adapter_ref
from rows_ref import check

pytestmark = pytest.mark.gpu

TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


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


def randn(torch, seed, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(getattr(torch, dtype))


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


class Case:
    """Inputs of a call; T rows, of which the documents may cover fewer."""

    def __init__(self, torch, dtype, wtype, lens, ids, n, r, K, N, T=None, base=True, seed=1, scale=1.5):
        self.cu, self.ids, self.scale = offsets(lens), ids, scale
        T = int(self.cu[-1]) if T is None else T
        self.x, self.dy = randn(torch, seed, dtype, T, K), randn(torch, seed + 1, dtype, T, N)
        self.a, self.b = randn(torch, seed + 2, wtype, n, r, K) * K ** -0.5, randn(torch, seed + 3, wtype, n, N, r) * r ** -0.5
        self.base = randn(torch, seed + 4, dtype, T, N) if base else None
        self.dx_base = randn(torch, seed + 5, dtype, T, K) if base else None

    def forward(self, nxg, **kw):
        return nxg.adapter_rows(self.x, self.a, self.b, self.cu, self.ids, self.scale, base=self.base, **kw)

    def backward(self, nxg, s, **kw):
        return nxg.adapter_rows_backward(self.dy, self.x, self.a, self.b, s, self.cu, self.ids, self.scale, base=self.dx_base, **kw)

    def check(self, nxg, torch):
        y, s = self.forward(nxg)
        n = int(self.cu[-1])
        (ry, by), (rs, bs) = adapter_ref.adapter(self.x, self.a, self.b, self.cu, self.ids, self.scale, self.base)
        check("y", y[:n], ry[:n], by[:n])
        check("s", s[:n], rs[:n], bs[:n])
        grads = self.backward(nxg, s)
        ref = adapter_ref.adapter_back(self.dy, self.x, self.a, self.b, s, self.cu, self.ids, self.scale, self.dx_base)
        check("dx", grads[0][:n], ref[0][0][:n], ref[0][1][:n])
        check("da", grads[1], *ref[1])
        check("db", grads[2], *ref[2])
        return (y, s) + grads


MIXED = [5, 0, 40, 1, 130, 17, 0, 64, 33]
MIXED_IDS = [2, 0, 0, 3, 2, -1, 1, 0, 7]        # of 5: 1 has no rows, 4 no document, -1 and 7 are none


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("r", [1, 4, 8, 16, 17, 32, 40, 64, 65, 128])
def test_ranks(nxg, torch, dev, dtype, wtype, r):
    say(f"adapter_rows {dtype} {wtype} r={r}")
    Case(torch, dtype, wtype, MIXED, MIXED_IDS, 5, r, 192, 320).check(nxg, torch)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (7, 65), (1024, 24), (24, 1024), (1023, 130), (520, 1000)])
def test_widths(nxg, torch, dev, dtype, wtype, K, N):
    say(f"adapter_rows {dtype} {wtype} K={K} N={N}")
    for r, base in ((16, True), (33, False)):
        Case(torch, dtype, wtype, MIXED, MIXED_IDS, 5, r, K, N, base=base).check(nxg, torch)


@pytest.mark.parametrize("lens,ids,n", [
    ([1], [0], 1), ([1], [-1], 1), ([0], [0], 2), ([2], [1], 2), ([3000], [0], 1), ([1] * 64, [i % 64 for i in range(64)], 64),
    ([1] * 300, [i % 3 for i in range(300)], 3), ([1] * 5000, [(i * 7) % 11 - 1 for i in range(5000)], 10),
    ([20, 1500, 3, 700, 0, 900] * 3, [0, 1, 1, 0, 1, 2] * 3, 4), ([3] * 200, [i for i in range(200)], 1200)],
    ids=["1", "none", "empty", "2", "3000", "64x1", "300x1", "5000x1", "mixed", "1200adapters"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_documents(nxg, torch, dev, dtype, lens, ids, n):
    say(f"adapter_rows {dtype} {len(lens)} documents, {n} adapters")
    Case(torch, dtype, dtype, lens, ids, n, 8, 128, 72).check(nxg, torch)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("r", [16, 64, 128])
def test_many_rows(nxg, torch, dev, dtype, wtype, r):
    """Tiles of 64 rows, several chunks an adapter; the same call gives the same bits."""
    say(f"adapter_rows {dtype} {wtype} r={r}, 33,000 rows")
    c = Case(torch, dtype, wtype, [20000, 13, 12000, 987], [1, 0, 1, -1], 3, r, 64, 136, T=33100)
    first = c.check(nxg, torch)
    y, s = c.forward(nxg)
    assert all(torch.equal(a[:33000], b[:33000]) for a, b in zip(first[:3], (y, s, c.backward(nxg, first[1])[0])))
    assert all(torch.equal(a, b) for a, b in zip(first[3:], c.backward(nxg, first[1])[1:]))


@pytest.mark.parametrize("dtype,wtype", TYPES)
def test_rows_behind_the_documents(nxg, torch, dev, dtype, wtype):
    say(f"adapter_rows {dtype} {wtype} rows behind the documents, in place, strided")
    T, K, N, r = 200, 64, 72, 16
    c = Case(torch, dtype, wtype, [50, 30, 70], [1, -1, 0], 2, r, K, N, T=T)
    y, s = c.forward(nxg)
    want = (y, s) + c.backward(nxg, s)
    for off in (0, 3):                                            # 3: rows off 16 bytes
        wide = lambda t: torch.full((T, t.shape[1] + 16), 7.0, dtype=t.dtype, device="cuda")[:, off:off + t.shape[1]]  # noqa: E731
        d = Case(torch, dtype, wtype, [50, 30, 70], [1, -1, 0], 2, r, K, N, T=T)
        for name in ("x", "dy", "base", "dx_base"):
            t = wide(getattr(c, name))
            t.copy_(getattr(c, name))
            setattr(d, name, t)
        out, s_out, dx = wide(c.base), torch.full((T, r), 7.0, device="cuda"), wide(c.x)
        d.forward(nxg, out=out, s=s_out)
        grads = d.backward(nxg, s_out, dx=dx)
        for got, ref in zip((out, s_out, dx), want):
            if off == 0:                                          # the single-value path sums in the same order
                assert torch.equal(got[:150], ref[:150])
            assert (got[150:] == 7).all()
        d.check(nxg, torch)
        assert all(torch.equal(a, b) for a, b in zip(grads[1:], want[3:])) or off
        # over the base
        at, dat = d.base.clone(), d.dx_base.clone()
        kept, dkept = d.base, d.dx_base
        d.base, d.dx_base = wide(at), wide(dat)
        d.base.copy_(at)
        d.dx_base.copy_(dat)
        d.forward(nxg, out=d.base, s=s_out)
        d.backward(nxg, s_out, dx=d.dx_base)
        assert torch.equal(d.base[:150], out[:150]) and torch.equal(d.base[150:], kept[150:])
        assert torch.equal(d.dx_base[:150], dx[:150]) and torch.equal(d.dx_base[150:], dkept[150:])


def test_shared_rows(nxg, torch, dev):
    """A row for all tokens (a stride of 0) as x, dy and base."""
    say("adapter_rows broadcast rows")
    c = Case(torch, "bfloat16", "bfloat16", [40, 25], [0, 1], 2, 16, 64, 64)
    for name in ("x", "dy", "base", "dx_base"):
        setattr(c, name, getattr(c, name)[:1].expand(65, 64))
    c.check(nxg, torch)


@pytest.mark.parametrize("dtype,wtype", [("float32", "bfloat16"), ("float16", "float16"), ("bfloat16", "bfloat16")])
def test_values_that_are_not_finite_stay_in_their_rows(nxg, torch, dev, dtype, wtype):
    """Rows with an infinity or a NaN, in a tile and a chunk with others: forward and dx of other rows do not change, nor the
    gradients of other adapters; a row of no adapter has no part at all."""
    say(f"adapter_rows {dtype} not finite")
    lens, ids = [30, 40, 50], [0, 1, -1]
    c = Case(torch, dtype, wtype, lens, ids, 2, 16, 64, 64)
    y, s = c.forward(nxg)
    want = (y, s) + c.backward(nxg, s)
    z = Case(torch, dtype, wtype, lens, ids, 2, 16, 64, 64)
    z.x[3, 5], z.dy[4, 7], z.base[6, 1] = math.inf, math.nan, math.nan
    z.x[100], z.dy[100] = math.nan, math.inf
    y, s = z.forward(nxg)
    got = (y, s) + z.backward(nxg, s)
    for name, g, w, bad in zip(("y", "s", "dx"), got, want, ((3, 6), (3,), (4,))):
        keep = [i for i in range(120) if i not in bad]
        assert torch.equal(g[keep], w[keep]), name
    assert not torch.isfinite(got[0][3]).any() and not torch.isfinite(got[2][4]).any()
    assert torch.isnan(got[0][6, 1]) and torch.equal(got[0][6, 2:], want[0][6, 2:])
    for g, w in zip(got[3:], want[3:]):
        assert torch.equal(g[1], w[1]) and not torch.isfinite(g[0]).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_large_and_small_values(nxg, torch, dev, dtype):
    """s and g past fp16's range and below its steps: they are carried in wider types."""
    say(f"adapter_rows {dtype} large and small values")
    c = Case(torch, dtype, dtype, [70, 30], [0, 1], 2, 16, 256, 128, scale=2.0 ** -12)
    c.x *= 512.0
    c.a *= 256.0
    c.dy[:40] *= 2.0 ** -10
    c.b *= 2.0 ** -4
    (_, s) = c.forward(nxg)
    assert float(s.abs().max()) > 65504.0
    c.check(nxg, torch)


def test_gradients_against_differences(nxg, torch, dev):
    say("adapter_rows gradients against differences")
    c = Case(torch, "float32", "float32", [6, 5], [1, 0], 2, 4, 24, 16)
    _, s = c.forward(nxg)
    grads = c.backward(nxg, s)
    f = lambda x, a, b: float((adapter_ref.adapter(x, a, b, c.cu, c.ids, c.scale, None)[0][0] * c.dy.double()).sum())  # noqa: E731
    args = [c.x.double(), c.a.double(), c.b.double()]
    for i, grad in enumerate(grads):
        grad = grad.double() - (c.dx_base.double() if i == 0 else 0.0)
        step = torch.sign(randn(torch, 9 + i, "float32", *args[i].shape)).double() * 2.0 ** -16
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step, args[i] - step
        diff = (f(*up) - f(*down)) / 2
        want = float((grad * step).sum())
        # fp32 roundings of the gradient and of dx's base (2^-18 of their sizes is far above them); the map is linear in each
        size = grad.abs() + (c.dx_base.double().abs() if i == 0 else 0.0)
        assert abs(diff - want) <= 2.0 ** -18 * float((size * step.abs()).sum()), (i, diff, want)


def test_rows_far_apart(nxg, torch, dev):
    """Rows over more than 4 GiB."""
    say("adapter_rows far apart")
    T, C, stride = 130, 64, 20_000_000
    buf = torch.empty((T - 1) * stride + 6 * C, dtype=torch.bfloat16, device="cuda")
    c = Case(torch, "bfloat16", "bfloat16", [100, 30], [1, 0], 2, 16, C, C)
    for i, name in enumerate(("x", "dy", "base", "dx_base")):
        t = buf.as_strided((T, C), (stride, 1), i * C)
        t.copy_(getattr(c, name))
        setattr(c, name, t)
    y, s = c.forward(nxg, out=buf.as_strided((T, C), (stride, 1), 4 * C))
    dx = c.backward(nxg, s, dx=buf.as_strided((T, C), (stride, 1), 5 * C))[0]
    d = Case(torch, "bfloat16", "bfloat16", [100, 30], [1, 0], 2, 16, C, C)
    want = d.check(nxg, torch)
    assert torch.equal(y, want[0]) and torch.equal(dx, want[2])


def test_offsets_and_ids_of_the_device(nxg, torch, dev):
    """Device offsets and ids; offsets that do not rise, and ids of no adapter, write nothing past their rows."""
    say("adapter_rows device offsets, bad ones")
    c = Case(torch, "bfloat16", "bfloat16", MIXED, MIXED_IDS, 5, 16, 64, 64)
    want = c.check(nxg, torch)
    cu, ids = (torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda") for v in (c.cu, c.ids))
    host = c.cu, c.ids
    c.cu, c.ids = cu, ids
    y, s = c.forward(nxg)
    assert all(torch.equal(a, b) for a, b in zip((y, s) + c.backward(nxg, s), want))
    T = int(host[0][-1])
    for bad in ([0, T, 0, T, 0, T, 0, T, 0, T], [T, 5, 3, 2, 1, 1, 1, 1, 1, 0], [-5, -1, 2 ** 31 - 1, -2 ** 31, 7, 7, 900, 3, 5, 10000],
                [T - 1] * 10):
        c.cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        guard = torch.full((T + 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        n = nxg.adapter_rows_backward_workspace_bytes(c.x, c.a, c.b, c.cu, c.ids)
        ws = torch.full((n + 64,), 7, dtype=torch.uint8, device="cuda")
        y, s = c.forward(nxg, out=guard[1:T + 1])
        c.backward(nxg, torch.nan_to_num(s), dx=guard[1:T + 1], workspace=ws[:n])
        assert (guard[0] == 7).all() and (guard[-1] == 7).all() and (ws[n:] == 7).all()
    with pytest.raises(ValueError, match="ids"):
        nxg.adapter_rows(c.x, c.a, c.b, host[0], [0, 1])
    with pytest.raises(ValueError, match="ids"):
        nxg.adapter_rows(c.x, c.a, c.b, host[0], ids.long())


def test_no_rows(nxg, torch, dev):
    say("adapter_rows no rows")
    c = Case(torch, "bfloat16", "bfloat16", [0, 0], [0, 1], 3, 16, 64, 64)
    y, s = c.forward(nxg)
    dx, da, db = c.backward(nxg, s)
    assert y.shape == (0, 64) and dx.shape == (0, 64) and (da == 0).all() and (db == 0).all()


def test_refusals_of_the_python_side(nxg, torch, dev):
    say("adapter_rows refusals")
    c = Case(torch, "bfloat16", "bfloat16", [40], [0], 2, 16, 64, 64)
    _, s = c.forward(nxg)
    n = nxg.adapter_rows_backward_workspace_bytes(c.x, c.a, c.b, c.cu, c.ids)
    with pytest.raises(ValueError, match="workspace"):
        c.backward(nxg, s, workspace=torch.empty(n - 16, dtype=torch.uint8, device="cuda"))
    for kw in ({"out": c.x[:, :8]}, {"out": c.x.float()}, {"s": s.half()}, {"s": s[:, :8]}, {"out": c.x}):
        with pytest.raises(ValueError):
            c.forward(nxg, **kw)
    for kw in ({"dx": c.dy}, {"da": c.b}, {"db": c.b}, {"da": c.a.float()}):
        with pytest.raises(ValueError):
            c.backward(nxg, s, **kw)
    with pytest.raises(ValueError, match="type"):
        nxg.adapter_rows(c.x, c.a.half(), c.b.half(), c.cu, c.ids)
    with pytest.raises(ValueError, match="fit"):
        nxg.adapter_rows(c.x[:, :32], c.a, c.b, c.cu, c.ids)
    with pytest.raises(ValueError, match="contiguous"):
        nxg.adapter_rows(c.x, c.a.transpose(1, 2), c.b, c.cu, c.ids)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("r,n", [(16, 1), (128, 5)])
def test_single_rows_that_share_adapters(nxg, torch, dev, dtype, wtype, r, n):
    """Requests of one row go together by their adapters, beside empty and longer ones: the same bits as one by one."""
    say(f"adapter_rows {dtype} {wtype} r={r}, requests of one row, {n} adapters")
    lens = [1] * 70 + [0, 0, 0, 17, 1, 1, 0] + [1] * 200 + [0] * 40
    ids = [(7 * i + i // 13) % (n + 1) - 1 if i % 5 else 0 for i in range(len(lens))]
    assert sum(lens) <= len(lens) and len(lens) > n
    c = Case(torch, dtype, wtype, lens, ids, n, r, 320, 136)
    y, s = c.check(nxg, torch)[:2]
    for d in (0, 1, 69, 73, 74, 100, 260):
        rows = slice(int(c.cu[d]), int(c.cu[d + 1]))
        one, s_one = nxg.adapter_rows(c.x[rows], c.a, c.b, [0, lens[d]], [ids[d]], c.scale, base=c.base[rows])
        assert torch.equal(one, y[rows]) and torch.equal(s_one, s[rows]), d
