"""GPU: attention_rows and attention_rows_backward against 64 bits (rows_ref.py, with the bounds of their
roundings): types, head sizes and ratios, packed documents of one token to more than a tile, empty
documents, windows that leave rows without a key, few queries over many keys, strides, rows behind the
last document."""
from __future__ import annotations

import math

import numpy as np
import pytest

import rows_ref

pytestmark = pytest.mark.gpu


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


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def make(torch, dtype, lens, keys, H, G, D, seed, grad=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    T, K = sum(lens), sum(keys)
    return (rnd(T, H, D).to(dtype), rnd(K, G, D).to(dtype), rnd(K, G, D).to(dtype), (grad * rnd(T, H, D)).to(dtype))


def run_and_check(nxg, torch, dtype, lens, keys=None, H=4, G=2, D=64, left=-1, right=-1, scale=None, seed=0, inputs=None, grad=True):
    keys = keys or lens
    q, k, v, do = inputs or make(torch, dtype, lens, keys, H, G, D, seed)
    cu_q, cu_k = offsets(lens), offsets(keys)
    kw = dict(left=left, right=right, scale=scale)
    out, lse = nxg.attention_rows(q, k, v, cu_q, cu_k, **kw)
    ref = rows_ref.attention(q, k, v, cu_q, cu_k, 1 / math.sqrt(D) if scale is None else scale, left, right, do if grad else None)
    rows_ref.check("out", out, *ref["out"])
    rows_ref.check("lse", lse, *ref["lse"])
    if grad:
        for name, t in zip(("dq", "dk", "dv"), nxg.attention_rows_backward(do, q, k, v, out, lse, cu_q, cu_k, **kw)):
            rows_ref.check(name, t, *ref[name])
    return q, k, v, do, out, lse


TYPES = ["bfloat16", "float16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 128])
def test_head_sizes(nxg, torch, dev, dtype, D):
    say(f"attention_rows {dtype} D={D}")
    run_and_check(nxg, torch, getattr(torch, dtype), [70, 1, 33], D=D, right=0, seed=D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G", [(1, 1), (2, 2), (8, 1), (6, 2), (16, 8), (12, 4), (40, 1), (129, 1)])
def test_head_ratios(nxg, torch, dev, dtype, H, G):
    say(f"attention_rows {dtype} H={H} G={G}")
    run_and_check(nxg, torch, getattr(torch, dtype), [5, 77, 2], H=H, G=G, right=0, seed=H)


WINDOWS = [(-1, -1), (-1, 0), (0, 0), (5, 5), (64, 64), (100, 0), (0, 70), (-1, 3), (3, -1)]


@pytest.mark.parametrize("left,right", WINDOWS)
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [128, 64, 65], [300, 17, 1, 129]], ids=str)
def test_windows(nxg, torch, dev, lens, left, right):
    say(f"attention_rows lens={lens} window={left},{right}")
    run_and_check(nxg, torch, torch.bfloat16, lens, left=left, right=right, seed=len(lens))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("left,right", [(-1, -1), (-1, 0), (20, 20), (0, 0)])
def test_long_document(nxg, torch, dev, dtype, left, right):
    say(f"attention_rows {dtype} 1500 tokens, window={left},{right}")
    run_and_check(nxg, torch, getattr(torch, dtype), [1500, 700], H=2, G=1, left=left, right=right, seed=3)


@pytest.mark.parametrize("lens,keys", [([1], [1000]), ([1, 1, 1], [5, 3000, 64]), ([3, 7], [500, 2]), ([200, 5], [9, 130]),
                                       ([4, 4, 4], [0, 10, 0]), ([0, 5, 0, 9], [7, 5, 0, 200])], ids=str)
@pytest.mark.parametrize("left,right", [(-1, -1), (-1, 0), (10, 0), (2, 2)])
def test_other_keys(nxg, torch, dev, lens, keys, left, right):
    """Queries and keys of different lengths: more queries than keys leave the first rows of a causal
    document without a key, documents without keys all of theirs."""
    say(f"attention_rows lens={lens} keys={keys} window={left},{right}")
    run_and_check(nxg, torch, torch.bfloat16, lens, keys, left=left, right=right, seed=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_few_queries_split(nxg, torch, dev, dtype, D):
    """One query over many keys: the keys shared out over workgroups, joined afterwards; without a workspace
    one workgroup takes them all."""
    say(f"attention_rows {dtype} 1 query over 20,000 keys D={D}")
    dt = getattr(torch, dtype)
    q, k, v, _, out, lse = run_and_check(nxg, torch, dt, [1], [20000], H=4, G=2, D=D, seed=D, grad=False)
    import ctypes
    p = nxg.rows._AttentionParams(nxg.rows._type_of(q, "q"), 4, 2, D, 1, 20000, 1, None, None, -1, -1, 1.0)
    assert nxg.load_library().nxg_attention_rows_workspace_bytes(ctypes.byref(p)) > 0, "this launch is to be split"
    small = torch.empty(16, dtype=torch.uint8, device="cuda")
    out2, lse2 = nxg.attention_rows(q, k, v, offsets([1]), offsets([20000]), workspace=small)
    ref = rows_ref.attention(q, k, v, offsets([1]), offsets([20000]), 1 / math.sqrt(D), -1, -1)
    rows_ref.check("out", out2, *ref["out"])
    rows_ref.check("lse", lse2, *ref["lse"])


def test_many_small_documents(nxg, torch, dev):
    """More documents than are tried at a time, among them empty ones."""
    say("attention_rows 700 documents")
    rng = np.random.default_rng(0)
    lens = [int(n) for n in rng.integers(0, 4, 700)]
    run_and_check(nxg, torch, torch.bfloat16, lens, H=2, G=1, D=32, right=0)


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_scores(nxg, torch, dev, dtype):
    """Scores of up to +-2,000 (one key has all the weight) and of a tiny scale (all alike), rising along
    the keys so that the running maximum moves in every tile."""
    say(f"attention_rows {dtype} extreme scores")
    dt = getattr(torch, dtype)
    q, k, v, do = make(torch, dt, [200], [200], 2, 1, 64, 5)
    ramp = torch.linspace(0.1, 6, 200, device="cuda")[:, None, None]
    k2 = (k.abs() * ramp).to(dt)
    q2 = q.abs()
    run_and_check(nxg, torch, dt, [200], H=2, G=1, scale=2.0, inputs=(q2, k2, v, do))
    run_and_check(nxg, torch, dt, [200], H=2, G=1, scale=2.0, inputs=((-q2), k2, v, do))
    run_and_check(nxg, torch, dt, [200], H=2, G=1, scale=1e-6, inputs=(q, k, v, do))


@pytest.mark.parametrize("grad", [1e-4, 300.0])
def test_fp16_gradient_range(nxg, torch, dev, grad):
    """fp16: upstream gradients so small or large that dS itself would leave the type's range."""
    say(f"attention_rows fp16 dout of {grad}")
    q, k, v, do = make(torch, torch.float16, [900], [900], 2, 1, 64, 7, grad)
    run_and_check(nxg, torch, torch.float16, [900], H=2, G=1, inputs=(q, k, v, do))


@pytest.mark.parametrize("layout", ["fused", "heads", "wide", "broadcast"])
def test_strides(nxg, torch, dev, layout):
    say(f"attention_rows layout {layout}")
    lens, H, G, D = [90, 3, 40], 4, 2, 64
    T = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    if layout == "fused":
        rows = rnd(T, H + 2 * G, D)
        q, k, v, do = rows[:, :H], rows[:, H:H + G], rows[:, H + G:], rnd(T, H, D)
    elif layout == "heads":
        q, k, v, do = (rnd(n, T, D).transpose(0, 1) for n in (H, G, G, H))
    elif layout == "wide":
        q, k, v, do = (rnd(T + 2, n + 3, D + 24)[1:T + 1, 2:n + 2, 8:D + 8] for n in (H, G, G, H))
    else:                         # one head's rows for all, one row for all keys
        q, do = rnd(T, 1, D).expand(T, H, D), rnd(1, H, D).expand(T, H, D)
        k, v = rnd(T, 1, D).expand(T, G, D), rnd(1, G, D).expand(T, G, D)
    cu = offsets(lens)
    ref = rows_ref.attention(q, k, v, cu, cu, 0.125, -1, 0, do)
    # outputs with strides of their own, in memory that nothing else of may change
    base = [torch.full((T + 2, n + 1, D + 8), 7.0, dtype=torch.bfloat16, device="cuda") for n in (H, H, G, G)]
    out, dq, dk, dv = (b[1:T + 1, :b.shape[1] - 1, :D] for b in base)
    o, lse = nxg.attention_rows(q, k, v, cu, left=-1, right=0, out=out)
    nxg.attention_rows_backward(do, q, k, v, o, lse, cu, left=-1, right=0, dq=dq, dk=dk, dv=dv)
    for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        rows_ref.check(name, t, *ref[name])
    for b in base:
        n = b.shape[1] - 1
        assert (b[0] == 7).all() and (b[-1] == 7).all() and (b[:, n] == 7).all() and (b[:, :, D:] == 7).all()


def test_rows_outside_documents_are_left(nxg, torch, dev):
    say("attention_rows rows outside the documents")
    H, G, D = 4, 2, 64
    q, k, v, do = make(torch, torch.bfloat16, [100], [120], H, G, D, 4)
    for t in (q, do):
        t[80:] = math.nan
        t[:3] = math.inf
    for t in (k, v):
        t[90:] = math.nan
        t[:5] = math.inf
    cu_q, cu_k = np.array([3, 40, 40, 80], np.int32), np.array([5, 30, 31, 90], np.int32)
    ref = rows_ref.attention(q, k, v, cu_q, cu_k, 0.125, -1, -1, do)
    out, lse = torch.full_like(q, 7), torch.full((100, H), 7.0, device="cuda")
    grads = [torch.full_like(t, 7) for t in (q, k, v)]
    nxg.attention_rows(q, k, v, cu_q, cu_k, out=out, lse=lse)
    nxg.attention_rows_backward(do, q, k, v, out, lse, cu_q, cu_k, dq=grads[0], dk=grads[1], dv=grads[2])
    for name, t, a, b in (("out", out, 3, 80), ("lse", lse, 3, 80), ("dq", grads[0], 3, 80), ("dk", grads[1], 5, 90), ("dv", grads[2], 5, 90)):
        rows_ref.check(name, t[a:b], ref[name][0][a:b], ref[name][1][a:b])
        assert (t[:a] == 7).all() and (t[b:] == 7).all(), name


def test_nothing_to_do(nxg, torch, dev):
    say("attention_rows of no rows")
    e = lambda n: torch.empty(0, n, 64, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    out, lse = nxg.attention_rows(e(4), e(2), e(2), [0, 0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    dq, dk, dv = nxg.attention_rows_backward(e(4), e(4), e(2), e(2), out, lse, [0, 0])
    assert dq.numel() == dk.numel() == dv.numel() == 0
    # queries without any key, keys without any query
    q, k, v, do = make(torch, torch.bfloat16, [5], [5], 4, 2, 64, 1)
    out, lse = nxg.attention_rows(q, e(2), e(2), [0, 5], [0, 0])
    assert (out == 0).all() and (lse == -math.inf).all()
    assert (nxg.attention_rows_backward(do, q, e(2), e(2), out, lse, [0, 5], [0, 0])[0] == 0).all()
    out, lse = nxg.attention_rows(e(4), k, v, [0, 0], [0, 5])
    _, dk, dv = nxg.attention_rows_backward(e(4), e(4), k, v, out, lse, [0, 0], [0, 5])
    assert (dk == 0).all() and (dv == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_again(nxg, torch, dev, dtype):
    say(f"attention_rows {dtype} twice")
    dt = getattr(torch, dtype)
    lens = [513, 40, 1]
    q, k, v, do = make(torch, dt, lens, lens, 8, 2, 64, 9)
    cu = offsets(lens)
    a = [t for t in nxg.attention_rows(q, k, v, cu, right=0)]
    a += nxg.attention_rows_backward(do, q, k, v, a[0], a[1], cu, right=0)
    b = [t for t in nxg.attention_rows(q, k, v, cu, right=0)]
    b += nxg.attention_rows_backward(do, q, k, v, b[0], b[1], cu, right=0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_against_differences(nxg, torch, dev):
    """The gradient along random directions against (f(x + t d) - f(x - t d)) / 2t of the 64-bit forward pass."""
    say("attention_rows gradient against differences")
    lens, H, G, D = [40, 9], 4, 2, 64
    q, k, v, do = make(torch, torch.bfloat16, lens, lens, H, G, D, 11)
    cu = offsets(lens)
    out, lse = nxg.attention_rows(q, k, v, cu, right=0)
    grads = nxg.attention_rows_backward(do, q, k, v, out, lse, cu, right=0)
    f = lambda a, b, c: float((rows_ref.attention(a, b, c, cu, cu, 0.125, -1, 0)["out"][0] * do.double()).sum())  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(1)
    # rows_ref takes the type's bounds from its inputs' type: float32 ones here, exact for these values
    xs = [t.float() for t in (q, k, v)]
    for i, grad in enumerate(grads):
        step = torch.sign(torch.randn(xs[i].shape, device="cuda", generator=g)) * 2.0 ** -10
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + step, xs[i] - step
        diff = (f(*up) - f(*down)) / 2
        want = float((grad.double() * step.double()).sum())
        bound = float((rows_ref.attention(q, k, v, cu, cu, 0.125, -1, 0, do)[("dq", "dk", "dv")[i]][1] * step.double().abs()).sum())
        # the difference's own third-order term: 2^-20 of the values here
        assert abs(diff - want) <= bound + 2.0 ** -16, (i, diff, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,lens,at", [(4, 2, [70, 20], [69, 40]), (4, 2, [300], [0, 150, 299]), (16, 16, [2100], [1000, 2099])])
def test_forward_leaves_out_what_is_not_seen(nxg, torch, dev, dtype, H, G, lens, at):
    """NaN and infinities in keys and values: only the queries that see them feel them (few-pairs kernel,
    and 128 pairs a workgroup)."""
    say(f"attention_rows {dtype} {lens}: NaN and infinities at {at}")
    dt = getattr(torch, dtype)
    for left, right in ((-1, 0), (10, 0), (40, 40), (5, -1)):
        q, k, v, _ = make(torch, dt, lens, lens, H, G, 64, 3)
        for i, t in enumerate(at):
            v[t, :, i::7] = math.inf if i % 2 else math.nan
            if i % 2 == 0:
                k[t, :, 5] = math.nan
        run_and_check(nxg, torch, dt, lens, H=H, G=G, left=left, right=right, inputs=(q, k, v, None), grad=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", ["q", "k", "v", "dout"])
def test_gradients_leave_out_what_is_not_seen(nxg, torch, dev, dtype, D, bad):
    """A token's NaN (in one input) reaches the gradients of the tokens that it sees or that see it, and what
    those touch, and no others."""
    say(f"attention_rows_backward {dtype} D={D}: NaN in {bad}")
    dt = getattr(torch, dtype)
    lens = [150, 75]
    for left, right in ((-1, 0), (7, 7), (12, 0), (0, 3)):
        tensors = dict(zip(("q", "k", "v", "dout"), make(torch, dt, lens, lens, 4, 2, D, 5)))
        for t in (100, 149, 160):
            tensors[bad][t] = math.nan
        run_and_check(nxg, torch, dt, lens, H=4, G=2, D=D, left=left, right=right, inputs=tuple(tensors.values()))


@pytest.mark.parametrize("left,right", [(-1, -1), (-1, 0), (7, -1), (70, 70)])
@pytest.mark.parametrize("H,G,D,same", [(16, 16, 32, True), (32, 16, 64, False)])
def test_documents_of_mixed_lengths(nxg, torch, dev, left, right, H, G, D, same):
    """Documents enough for more workgroups than run at once, among them empty ones and many of one length:
    every tile of every one is done once, in whatever order. More queries than keys, and fewer."""
    say(f"attention_rows 61 documents H={H} G={G} D={D} window={left},{right}")
    rng = np.random.default_rng(9)
    lens = [0, 400, 1, 128, 128, 256, 0, 129, 127] + [int(n) for n in rng.integers(0, 200, 50)] + [300, 0]
    keys = lens if same else [int(n) for n in rng.integers(0, 260, len(lens))]
    run_and_check(nxg, torch, torch.bfloat16, lens, keys, H=H, G=G, D=D, left=left, right=right, seed=D)


@pytest.mark.parametrize("n", [63, 64, 65, 130])
def test_number_of_documents(nxg, torch, dev, n):
    """About as many documents as a wave has lanes, and more."""
    say(f"attention_rows {n} documents")
    run_and_check(nxg, torch, torch.float16, [(37 * i) % 150 for i in range(n)], H=16, G=16, D=32, right=0, seed=n)


@pytest.mark.parametrize("stride,lens", [(8_000_000, [250, 50]), (20_000_000, [130, 7])], ids=str)
@pytest.mark.parametrize("H,G", [(4, 2), (128, 128), (128, 64), (96, 32)])
def test_rows_far_apart(nxg, torch, dev, stride, lens, H, G):
    """Rows over more than 4 GiB: a tile's own offsets fit 32 bits, or do not either."""
    say(f"attention_rows H={H} G={G} rows {2 * stride} bytes apart")
    T, D = sum(lens), 64
    need = (T - 1) * stride + 4 * (H + G) * D
    buf = torch.empty(need, dtype=torch.bfloat16, device="cuda")
    at, views = 0, []
    for n in (H, H, H, H, G, G, G, G):
        views.append(buf.as_strided((T, n, D), (stride, D, 1), at))
        at += n * D
    q, do, out, dq, k, v, dk, dv = views
    g = torch.Generator(device="cuda").manual_seed(H)
    for t in (q, do, k, v):
        t.copy_(torch.randn(t.shape, device="cuda", generator=g))
    cu = offsets(lens)
    ref = rows_ref.attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, 0.125, -1, 0, do.contiguous())
    _, lse = nxg.attention_rows(q, k, v, cu, left=-1, right=0, out=out)
    nxg.attention_rows_backward(do, q, k, v, out, lse, cu, left=-1, right=0, dq=dq, dk=dk, dv=dv)
    for name, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        rows_ref.check(name, t, *ref[name])


@pytest.mark.parametrize("n,stride", [(1, 8_000_000), (1, 20_000_000), (3, 20_000_000)])
def test_few_queries_over_a_far_cache(nxg, torch, dev, n, stride):
    say(f"attention_rows {n} queries over keys {2 * stride} bytes apart")
    K, H, G, D = 600, 4, 2, 128
    buf = torch.empty((K - 1) * stride + 2 * G * D, dtype=torch.bfloat16, device="cuda")
    k, v = (buf.as_strided((K, G, D), (stride, D, 1), i * G * D) for i in range(2))
    g = torch.Generator(device="cuda").manual_seed(n)
    for t in (k, v):
        t.copy_(torch.randn(t.shape, device="cuda", generator=g))
    q = torch.randn(n, H, D, device="cuda", generator=g).bfloat16()
    out, lse = nxg.attention_rows(q, k, v, [0, n], [0, K], right=0)
    ref = rows_ref.attention(q, k.contiguous(), v.contiguous(), [0, n], [0, K], 1 / math.sqrt(D), -1, 0)
    rows_ref.check("out", out, *ref["out"])
    rows_ref.check("lse", lse, *ref["lse"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,D", [(8, 1, 96), (6, 2, 64), (5, 1, 128), (7, 1, 32)])
@pytest.mark.parametrize("lens,keys", [([900, 40, 0, 333], None), ([34, 1], [3000, 200]), ([1100, 9], [70, 0])], ids=str)
@pytest.mark.parametrize("left,right", [(-1, 0), (-1, -1), (200, 100)])
def test_gradients_of_few_long_documents(nxg, torch, dev, dtype, H, G, D, lens, keys, left, right):
    """Few tiles, each with much to go over: shared out over workgroups, for queries and for keys, documents of
    other lengths and shares that are empty among them."""
    say(f"attention_rows {dtype} H={H} G={G} D={D} lens={lens} keys={keys} window={left},{right}")
    run_and_check(nxg, torch, getattr(torch, dtype), lens, keys, H=H, G=G, D=D, left=left, right=right, seed=D)


def test_split_gradients_need_their_workspace(nxg, torch, dev):
    say("attention_rows_backward workspace of shares")
    q, k, v, do = make(torch, torch.bfloat16, [2000], [2000], 4, 1, 64, 3)
    n = nxg.rows.attention_rows_backward_workspace_bytes(q, k, v, [0, 2000], right=0)
    assert n > 4 * 2 * 2000 * 4 + 4 * 2 * 2000 * 64, "shares are left in the workspace"
    out, lse = nxg.attention_rows(q, k, v, [0, 2000], right=0)
    with pytest.raises(ValueError, match="workspace"):
        nxg.attention_rows_backward(do, q, k, v, out, lse, [0, 2000], right=0, workspace=torch.empty(n - 1, dtype=torch.uint8, device="cuda"))
    big = torch.full((n + 256,), 7, dtype=torch.uint8, device="cuda")
    a = nxg.attention_rows_backward(do, q, k, v, out, lse, [0, 2000], right=0, workspace=big[:n])
    assert (big[n:] == 7).all()
    b = nxg.attention_rows_backward(do, q, k, v, out, lse, [0, 2000], right=0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 80])
@pytest.mark.parametrize("n_docs", [40, 300])
def test_gradients_of_single_keys_cancel(nxg, torch, dev, dtype, D, n_docs):
    """A query of one key: dS = P (dP - delta) is 0, so that dQ and dK are what fp32 leaves of it, not what the rounding of
    `out` would. dP and delta: D products and sums each, off by D + 8 half steps of the sum of their sizes; P, whose
    exponent is rounded at up to 8 (2^-20 of it) and again by exp2, by 2^-18 at most, in both."""
    say(f"attention_rows {dtype} single keys D={D} {n_docs} documents")
    dt, H, G = getattr(torch, dtype), 4, 2
    for lens, keys, left, right in (([1] * n_docs, [1] * n_docs, -1, -1), ([3] * n_docs, [1] * n_docs, -1, -1), ([5] * n_docs, [5] * n_docs, 0, 0)):
        q, k, v, do = make(torch, dt, lens, keys, H, G, D, n_docs)
        cu_q, cu_k = offsets(lens), offsets(keys)
        out, lse = nxg.attention_rows(q, k, v, cu_q, cu_k, left=left, right=right)
        dq, dk, _ = nxg.attention_rows_backward(do, q, k, v, out, lse, cu_q, cu_k, left=left, right=right)
        at = torch.arange(len(q), device="cuda") if left == 0 else torch.arange(n_docs, device="cuda").repeat_interleave(lens[0])
        K, V = (t.double().repeat_interleave(H // G, 1)[at] for t in (k, v))      # of each query
        dO = do.double()
        e = 2.0 ** -17 * (dO * V).sum(2).abs() + 2 * (D + 8) * 2.0 ** -24 * (dO * V).abs().sum(2)
        least = rows_ref.least_step(dt)
        e = e[:, :, None] * 1.02 * D ** -0.5
        assert (dq.double().abs() <= e * K.abs() + least).all()
        b = torch.zeros(len(k), H, D, dtype=torch.float64, device="cuda").index_add_(0, at, e * q.double().abs())
        assert (dk.double().abs() <= b.reshape(len(k), G, H // G, D).sum(2) + least).all()
