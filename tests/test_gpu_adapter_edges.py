"""GPU: adapter_rows and adapter_rows_backward at the edges of their sizes: no rows, gradients inside other
tensors, many documents and adapters and the time they take."""
from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

from test_gpu_adapter_rows import Case

pytestmark = pytest.mark.gpu

TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"), ("float16", "float16"), ("bfloat16", "bfloat16")]


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.fixture(scope="module")
def dev(torch, nxg):
    nxg.init()
    return torch.device("cuda:0")


def guarded(torch, dtype, shape, lead):
    """A tensor of NaN inside a buffer of sevens, `lead` values behind the buffer's start."""
    n = 1
    for s in shape:
        n *= s
    buf = torch.full((n + lead + 64,), 7.0, dtype=dtype, device="cuda")
    t = buf[lead:lead + n].view(shape)
    t.fill_(float("nan"))
    return buf, t, slice(lead, lead + n)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("n_in,n_out", [(7, 64), (64, 7), (1, 1), (1023, 1023), (24, 40)])
@pytest.mark.parametrize("r", [4, 16, 65])
def test_gradients_of_no_rows(nxg, torch, dev, dtype, wtype, n_in, n_out, r):
    """Zeros for every value of da and db, nothing beside them: without rows (T = 0), and without documents (n_seqs = 0)."""
    print(f"adapter_rows_backward {dtype} {wtype} no rows, {n_in} to {n_out}, r={r}", flush=True)
    dt, wt, n = getattr(torch, dtype), getattr(torch, wtype), 3
    a, b = torch.ones(n, r, n_in, dtype=wt, device="cuda"), torch.ones(n, n_out, r, dtype=wt, device="cuda")
    for lead in (16, 17):                                       # on 16 bytes, and off them
        bufs = [guarded(torch, wt, t.shape, lead) for t in (a, b)]
        x, dy = (torch.empty(0, c, dtype=dt, device="cuda") for c in (n_in, n_out))
        nxg.adapter_rows_backward(dy, x, a, b, torch.empty(0, r, device="cuda"), [0, 0], [0], da=bufs[0][1], db=bufs[1][1])
        check(bufs)

        bufs = [guarded(torch, wt, t.shape, lead) for t in (a, b)]
        x, dy, s = (torch.ones(5, c, dtype=t, device="cuda") for c, t in ((n_in, dt), (n_out, dt), (r, torch.float32)))
        dx = torch.full_like(x, 7.0)
        types = {torch.float32: nxg.TYPE_F32, torch.float16: nxg.TYPE_F16, torch.bfloat16: nxg.TYPE_BF16}
        p = nxg.rows._adapter_params.pack(types[dt], types[wt], 5, n_in, n_out, r, n, 0, 0, 0, a.data_ptr(), b.data_ptr(), 1.0)
        L = nxg.load_library()
        ws = torch.empty(L.nxg_adapter_rows_backward_workspace_bytes(p), dtype=torch.uint8, device="cuda")
        rc = L.nxg_adapter_rows_backward(p, dy.data_ptr(), n_out, x.data_ptr(), n_in, s.data_ptr(), None, 0, dx.data_ptr(), n_in,
                                         bufs[0][1].data_ptr(), bufs[1][1].data_ptr(), ws.data_ptr(), ws.numel(),
                                         ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == nxg.NXG_OK
        check(bufs)
        assert (dx == 7).all()


def check(bufs):
    for buf, t, inside in bufs:
        assert (t == 0).all()
        assert (buf[:inside.start] == 7).all() and (buf[inside.stop:] == 7).all()


def single_rows(torch, dtype, n, r, S, extra=(), n_in=256, n_out=264):
    """Arguments of a call of S documents of one row of n adapters, and of documents of the `extra` lengths behind them."""
    g = torch.Generator(device="cuda").manual_seed(S)
    T = S + sum(extra)
    x, base = (torch.randn(T, c, device="cuda", generator=g).to(getattr(torch, dtype)) for c in (n_in, n_out))
    a, b = torch.randn(n, r, n_in, device="cuda", generator=g).to(x.dtype) / 16, torch.randn(n, n_out, r, device="cuda", generator=g).to(x.dtype)
    ids = torch.randint(-1, n, (S + len(extra),), device="cuda", dtype=torch.int32, generator=g)
    cu = torch.cumsum(torch.tensor([0] + [1] * S + list(extra), device="cuda"), 0).int()
    return x, a, b, cu, ids, 1.5, base


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("S,n", [(1023, 5), (1024, 300), (1025, 1), (5000, 300), (9001, 16), (20000, 3000), (40000, 70)])
def test_single_rows_gathered_or_not(nxg, torch, dev, dtype, S, n):
    """More rows than one search for an adapter's goes over: the same bits as in a call that takes every row by itself, which a longer
    document behind them makes of it."""
    print(f"adapter_rows {dtype} {S} documents of one row, {n} adapters", flush=True)
    x, a, b, cu, ids, scale, base = single_rows(torch, dtype, n, 16, S, (3,))
    y, s = nxg.adapter_rows(x[:S], a, b, cu[:S + 1], ids[:S], scale, base=base[:S])
    want, s_want = nxg.adapter_rows(x, a, b, cu, ids, scale, base=base)
    assert torch.equal(y, want[:S]) and torch.equal(s, s_want[:S])
    none = (ids[:S] < 0).nonzero()[:, 0]
    assert torch.equal(y[none], base[:S][none]) and (s[none] == 0).all()


def fastest(torch, call):
    best = float("inf")
    for _ in range(6):
        t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        t[0].record()
        call()
        t[1].record()
        torch.cuda.synchronize()
        best = min(best, t[0].elapsed_time(t[1]))
    return best


@pytest.mark.parametrize("dtype,r,n", [("float32", 16, 16), ("float32", 8, 64), ("bfloat16", 16, 16)])
def test_time_of_single_rows(nxg, torch, dev, dtype, r, n):
    """8 times the rows take about 8 times as long, not 64."""
    print(f"adapter_rows {dtype} r={r}: 4,096 and 32,768 documents of one row, {n} adapters", flush=True)
    ms = []
    for S in (4096, 32768):
        args = single_rows(torch, dtype, n, r, S)
        ms.append(fastest(torch, lambda: nxg.adapter_rows(*args[:6], base=args[6])))
    assert ms[1] < 12 * ms[0], ms


@pytest.mark.parametrize("dtype,r,T", [("bfloat16", 32, 32768), ("bfloat16", 64, 32768), ("bfloat16", 128, 65536), ("float32", 128, 65536)])
@pytest.mark.parametrize("length", [1, 6])
def test_time_of_short_documents(nxg, torch, dev, dtype, r, T, length):
    """A launch of many rows does not take a tile of 64 or 128 of them for every short document: 8 times the rows, about 8 times as long."""
    print(f"adapter_rows {dtype} r={r}: {T // 8} and {T} rows, {length} a document", flush=True)
    ms = []
    for rows in (T // 8, T):
        x, a, b, cu, ids, scale, base = single_rows(torch, dtype, 8, r, rows // length * length)
        cu, ids = cu[::length].contiguous(), ids[:rows // length]
        ms.append(fastest(torch, lambda: nxg.adapter_rows(x, a, b, cu, ids, scale, base=base)))
    assert ms[1] < 12 * ms[0], ms


@pytest.mark.parametrize("dtype,wtype", [("float32", "bfloat16"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("docs,n", [(64, 3), (65, 1), (1030, 700), (4096, 2), (4097, 40), (1000, 524), (1000, 525), (3, 5000)])
def test_many_documents(nxg, torch, dev, dtype, wtype, docs, n):
    """Documents of 0 to 6 rows of many adapters: of one wave and of all, prepared by one launch and by two."""
    print(f"adapter_rows {dtype} {wtype} {docs} documents of {n} adapters", flush=True)
    rng = random.Random(docs)
    lens, ids = [rng.randrange(7) for _ in range(docs)], [rng.randrange(-1, n + 1) if i % 3 else rng.randrange(min(n, 3)) for i in range(docs)]
    Case(torch, dtype, wtype, lens, ids, n, 8, 40, 24, T=sum(lens) + 5).check(nxg, torch)


def test_time_of_many_adapters(nxg, torch, dev):
    """Gradients of 4,096 documents with 1,000 adapters: what is done goes by the documents and the adapters, not by their product."""
    print("adapter_rows_backward, 4,096 documents of 4 rows, 10 and 1,000 adapters", flush=True)
    ms = []
    for n in (10, 1000):
        x, a, b, cu, ids, scale, _ = single_rows(torch, "bfloat16", n, 8, 16384, n_in=64, n_out=64)
        cu, ids = cu[::4].contiguous(), ids[:4096].clamp(min=0)
        dy, s = torch.ones_like(x), nxg.adapter_rows(x, a, b, cu, ids)[1]
        ms.append(fastest(torch, lambda: nxg.adapter_rows_backward(dy, x, a, b, s, cu, ids)))
    assert ms[1] < 4 * ms[0] + 0.1, ms


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_millions_of_documents(nxg, torch, dev, dtype):
    """As many documents as the header allows, nearly all of them empty: the same bits as without the empty ones."""
    S = (1 << 22) - 1
    print(f"adapter_rows {dtype} {S} documents", flush=True)
    x, a, b, _, _, scale, base = single_rows(torch, dtype, 5, 16, 600, n_in=64, n_out=72)
    at = torch.tensor([0, 3, 1000, 2_000_000, S - 1], device="cuda")             # documents of 120 rows each
    lens, ids = torch.zeros(S, dtype=torch.int64, device="cuda"), torch.full((S,), 4, dtype=torch.int32, device="cuda")
    lens[at], ids[at] = 120, torch.tensor([1, 0, -1, 1, 3], dtype=torch.int32, device="cuda")
    cu = torch.cat([lens.new_zeros(1), torch.cumsum(lens, 0)]).int()
    few = torch.arange(0, 601, 120, dtype=torch.int32, device="cuda")
    dy = torch.ones_like(base)
    for c, i in ((cu, ids), (few, ids[at].contiguous())):
        y, s = nxg.adapter_rows(x, a, b, c, i, scale, base=base)
        got = (y, s) + nxg.adapter_rows_backward(dy, x, a, b, s, c, i, scale)
        want = got if c is cu else want
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_ids_of_the_host(nxg, torch, dev):
    """Whole numbers of any kind, as cu_offsets takes them: lists, arrays and tensors; past 32 bits they are no adapter."""
    print("adapter_rows ids of the host", flush=True)
    x, a, b, _, _, scale, base = single_rows(torch, "bfloat16", 3, 8, 40, n_in=64, n_out=64)
    cu, ids = [0, 10, 15, 40], [2, 0, 1]
    want = nxg.adapter_rows(x, a, b, cu, ids, scale, base=base)
    kinds = [np.array(ids, t) for t in (np.uint8, np.int16, np.uint32, np.int64, np.uint64)]
    for host in kinds + [torch.tensor(ids, dtype=t) for t in (torch.uint8, torch.int16, torch.int32, torch.int64)] + \
            [torch.tensor([2, 9, 0, 9, 1, 9])[::2]]:
        got = nxg.adapter_rows(x, a, b, torch.tensor(cu), host, scale, base=base)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    far = nxg.adapter_rows(x, a, b, cu, np.array([2 ** 32, 2 ** 40 + 1, -2 ** 40]), scale, base=base)
    assert torch.equal(far[0], base) and (far[1] == 0).all()
    for bad in (torch.tensor([2.0, 0.0, 1.0]), torch.tensor(ids, dtype=torch.bfloat16), torch.tensor([True, False, True]), torch.tensor([[2, 0, 1]]), torch.tensor([2, 0]), [2.0, 0.0, 1.0], torch.tensor(ids, device="cuda")):
        with pytest.raises(ValueError, match="ids"):
            nxg.adapter_rows(x, a, b, cu, bad, scale, base=base)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("docs,n,rows", [(3000, 200, 1), (3000, 200, 3), (40, 5, 30)])
def test_replays_with_other_documents_and_adapters(nxg, torch, dev, dtype, docs, n, rows):
    """A captured call of many documents, replayed after its offsets and ids have changed, on another stream than it was made for:
    the bits of the same call made then."""
    print(f"adapter_rows {dtype} {docs} documents of {n} adapters, captured", flush=True)
    x, a, b, _, ids, scale, base = single_rows(torch, dtype, n, 8, docs * rows, n_in=64, n_out=72)
    cu = (torch.arange(docs + 1, device="cuda") * rows).int()
    ids, dy = ids[:docs].contiguous(), torch.ones_like(base)

    def both():
        y, s = nxg.adapter_rows(x, a, b, cu, ids, scale, base=base)
        return (y, s) + nxg.adapter_rows_backward(dy, x, a, b, s, cu, ids, scale)
    both()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = both()
    for turn in range(4):
        ids.copy_(torch.roll(ids, 1 + 7 * turn))
        if turn % 2:
            cu[docs // 3:docs // 2] = int(cu[docs // 3])             # empty ones, and a longer one behind them
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(u, v) for u, v in zip(got, both())), turn
