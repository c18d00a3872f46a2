"""GPU: qk_norm_rope_rows, its gradients and dropout_rows against 64 bits (adapter_ref.py, with the bounds of their roundings)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import adapter_ref
from rows_ref import check

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]
WTYPES = [("float32", "float32"), ("float16", "float32"), ("float16", "float16"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")]


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


def places(torch, lens):
    return torch.from_numpy(np.concatenate([np.arange(n) for n in lens] or [np.zeros(0)]).astype(np.int64)).cuda()


def freqs(nxg, torch, n):
    return torch.from_numpy(nxg.rope_frequencies(n, 10000.0)[0]).cuda()


def check_both(nxg, torch, q, k, wq, wk, f, lens, layout="half", mscale=1.0, eps=1e-6, outs=(None, None), **kw):
    pos = places(torch, lens)
    cu = offsets(lens)
    got = nxg.qk_norm_rope_rows(q, k, wq, wk, f, cu, eps=eps, layout=layout, mscale=mscale, q_out=outs[0], k_out=outs[1])
    check("q", got[0], *adapter_ref.qk_norm_rope(q, wq, f, pos, layout, mscale, eps))
    check("k", got[1], *adapter_ref.qk_norm_rope(k, wk, f, pos, layout, mscale, eps))
    dq_out, dk_out = randn(torch, 91, str(q.dtype)[6:], *q.shape), randn(torch, 92, str(q.dtype)[6:], *k.shape)
    grads = nxg.qk_norm_rope_rows_backward(dq_out, dk_out, q, k, wq, wk, f, cu, eps=eps, layout=layout, mscale=mscale)
    for name, i, dy, x, w in (("q", 0, dq_out, q, wq), ("k", 1, dk_out, k, wk)):
        dx, dw = adapter_ref.qk_norm_rope_back(dy, x, w, f, pos, layout, mscale, eps)
        check("d" + name, grads[i], *dx)
        check("dw" + name, grads[2 + i], *dw)
    return got, grads


@pytest.mark.parametrize("dtype,wtype", WTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,n", [(64, 64), (64, 32), (128, 128), (80, 40), (96, 96), (6, 2), (2, 2), (63, 20), (257, 128)])
def test_qk_norm_rope(nxg, torch, dev, dtype, wtype, layout, D, n):
    say(f"qk_norm_rope_rows {dtype} {wtype} {layout} D={D} n={n}")
    lens = [1, 40, 0, 3, 37]
    q, k = randn(torch, D, dtype, sum(lens), 5, D) * 2, randn(torch, D + 1, dtype, sum(lens), 2, D)
    wq, wk = randn(torch, 3, wtype, D), randn(torch, 4, wtype, D)
    check_both(nxg, torch, q, k, wq, wk, freqs(nxg, torch, n), lens, layout, 1.25)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D", [512, 1000, 1024, 1023])
def test_qk_large_heads(nxg, torch, dev, dtype, layout, D):
    say(f"qk_norm_rope_rows {dtype} {layout} D={D}")
    q, k = randn(torch, 1, dtype, 9, 2, D), randn(torch, 2, dtype, 9, 1, D)
    check_both(nxg, torch, q, k, randn(torch, 3, dtype, D), randn(torch, 4, dtype, D), freqs(nxg, torch, D // 4 * 2), [4, 5], layout)


def test_qk_sizes(nxg, torch, dev):
    say("qk_norm_rope_rows one token, many heads, many tokens, no tokens")
    f, w = freqs(nxg, torch, 64), randn(torch, 1, "float32", 64)
    for T, H, G, lens in ((1, 1, 1, [1]), (1, 300, 7, [1]), (2000, 3, 3, [1] * 1500 + [0, 500]), (9000, 16, 8, [9000])):
        q, k = randn(torch, T, "bfloat16", T, H, 64), randn(torch, T + 1, "bfloat16", T, G, 64)
        got, grads = check_both(nxg, torch, q, k, w, w + 1, f, lens)
    again = nxg.qk_norm_rope_rows_backward(got[0], got[1], q, k, w, w + 1, f, offsets(lens))
    assert all(torch.equal(a, b) for a, b in zip(again, nxg.qk_norm_rope_rows_backward(got[0], got[1], q, k, w, w + 1, f, offsets(lens))))
    none = nxg.qk_norm_rope_rows(q[:0], k[:0], w, w, f, [0, 0])
    assert none[0].shape == (0, 16, 64) and none[1].shape == (0, 8, 64)
    grads = nxg.qk_norm_rope_rows_backward(q[:0], k[:0], q[:0], k[:0], w, w, f, [0, 0])
    assert (grads[2] == 0).all() and (grads[3] == 0).all()


def test_qk_queries_alone_and_positions(nxg, torch, dev):
    say("qk_norm_rope_rows without keys, far positions")
    pos = torch.tensor([0, 1, -1, 65535, 1000003, 2 ** 31 - 1, -2 ** 31, 123456789], dtype=torch.int32, device="cuda")
    q, dy, w, f = randn(torch, 1, "float32", 8, 3, 64), randn(torch, 2, "float32", 8, 3, 64), randn(torch, 3, "float32", 64), freqs(nxg, torch, 32)
    out, none = nxg.qk_norm_rope_rows(q, None, w, None, f, positions=pos)
    assert none is None
    check("q", out, *adapter_ref.qk_norm_rope(q, w, f, pos.long(), "half", 1.0, 1e-6))
    dq, dk, dwq, dwk = nxg.qk_norm_rope_rows_backward(dy, None, q, None, w, None, f, positions=pos)
    assert dk is None and dwk is None
    dx, dw = adapter_ref.qk_norm_rope_back(dy, q, w, f, pos.long(), "half", 1.0, 1e-6)
    check("dq", dq, *dx)
    check("dwq", dwq, *dw)


def test_qk_turns_as_rope_rows(nxg, torch, dev):
    """A norm's weights of 1 over rows whose mean square is 1 leave rope_rows' result, within the norm's roundings."""
    say("qk_norm_rope_rows beside rope_rows")
    q = torch.sign(randn(torch, 1, "float32", 50, 4, 64))
    f, one = freqs(nxg, torch, 64), torch.ones(64, device="cuda")
    got = nxg.qk_norm_rope_rows(q, None, one, None, f, [0, 20, 50], eps=0.0)[0]
    assert float((got - nxg.rope_rows(q, f, [0, 20, 50])).abs().max()) <= 2 * (adapter_ref.RSTD + 6 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_qk_in_place_and_strides(nxg, torch, dev, dtype, layout):
    say(f"qk_norm_rope_rows {dtype} {layout} in place, strided")
    lens = [30, 11]
    T, D = sum(lens), 64
    f, wq, wk = freqs(nxg, torch, 32), randn(torch, 5, "float32", D), randn(torch, 6, "float32", D)
    rows, d_rows = randn(torch, 4, dtype, T, 9, D), randn(torch, 7, dtype, T, 9, D)
    q, k = rows[:, 1:6], rows[:, 6:8]
    dq, dk = d_rows[:, 1:6], d_rows[:, 6:8]
    want, _ = check_both(nxg, torch, q, k, wq, wk, f, lens, layout)
    grads = nxg.qk_norm_rope_rows_backward(dq, dk, q, k, wq, wk, f, offsets(lens), layout=layout)
    # rows that are not 16-byte aligned, and head-major ones
    odd = torch.zeros(T, 9, D + 1, dtype=rows.dtype, device="cuda")[:, :, 1:]
    odd.copy_(rows)
    check_both(nxg, torch, odd[:, 1:6], odd[:, 6:8], wq, wk, f, lens, layout)
    heads = rows.transpose(0, 1).contiguous().transpose(0, 1)
    to = torch.empty(9, T, D, dtype=rows.dtype, device="cuda").transpose(0, 1)
    check_both(nxg, torch, heads[:, 1:6], heads[:, 6:8], wq, wk, f, lens, layout, outs=(to[:, 1:6], to[:, 6:8]))
    # over the gradients, over the inputs, then forward over the inputs: the same bits, and nothing else written
    for over in ("gradients", "inputs"):
        x, g = rows.clone(), d_rows.clone()
        at = g if over == "gradients" else x
        keep = at.clone()
        got = nxg.qk_norm_rope_rows_backward(g[:, 1:6], g[:, 6:8], x[:, 1:6], x[:, 6:8], wq, wk, f, offsets(lens), layout=layout,
                                             dq=at[:, 1:6], dk=at[:, 6:8])
        assert all(torch.equal(a, b) for a, b in zip(got, grads)), over
        assert torch.equal(at[:, 0], keep[:, 0]) and torch.equal(at[:, 8], keep[:, 8])
    x = rows.clone()
    got = nxg.qk_norm_rope_rows(x[:, 1:6], x[:, 6:8], wq, wk, f, offsets(lens), layout=layout, q_out=x[:, 1:6], k_out=x[:, 6:8])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(x[:, 0], rows[:, 0]) and torch.equal(x[:, 8], rows[:, 8])


def test_qk_special_rows(nxg, torch, dev):
    """Zero rows, huge and tiny ones, a head with an infinity or a NaN: others do not change."""
    say("qk_norm_rope_rows special rows")
    x, w, f = randn(torch, 1, "float32", 8, 2, 64), randn(torch, 2, "float32", 64), freqs(nxg, torch, 64)
    x[1] = 0.0
    x[2] *= 1e15
    x[3] *= 1e-15
    pos = places(torch, [8])
    plain = nxg.qk_norm_rope_rows(x, None, w, None, f, [0, 8])[0]
    check("q", plain, *adapter_ref.qk_norm_rope(x, w, f, pos, "half", 1.0, 1e-6))
    z = x.clone()
    z[5, 0, 7], z[6, 1, 0] = math.inf, math.nan
    y = nxg.qk_norm_rope_rows(z, None, w, None, f, [0, 8])[0]
    keep = torch.ones(8, 2, dtype=torch.bool)
    keep[5, 0] = keep[6, 1] = False
    assert torch.equal(y[keep], plain[keep]) and torch.isnan(y[6, 1]).all() and torch.isnan(y[5, 0]).any()


def test_qk_gradient_against_differences(nxg, torch, dev):
    say("qk_norm_rope_rows gradient against differences")
    x, w, dy = randn(torch, 1, "float32", 6, 2, 64), randn(torch, 2, "float32", 64), randn(torch, 4, "float32", 6, 2, 64)
    f, pos = freqs(nxg, torch, 64), places(torch, [6])
    dx, _, dw, _ = nxg.qk_norm_rope_rows_backward(dy, None, x, None, w, None, f, [0, 6])
    fn = lambda *a: float((adapter_ref.qk_norm_rope(a[0], a[1], f, pos, "half", 1.0, 1e-6)[0] * dy.double()).sum())  # noqa: E731
    for i, grad in enumerate((dx, dw)):
        args = [x.double(), w.double()]
        step = torch.sign(randn(torch, 9 + i, "float32", *args[i].shape)).double() * 2.0 ** -16
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step, args[i] - step
        diff = (fn(*up) - fn(*down)) / 2
        want = float((grad.double() * step).sum())
        # fp32 roundings of the gradient (2^-18 of its size is far above them) and the third-order term
        assert abs(diff - want) <= 2.0 ** -18 * float((grad.double().abs() * step.abs()).sum()) + 2.0 ** -36, (i, diff, want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_qk_rows_far_apart(nxg, torch, dev, layout):
    """Rows over more than 4 GiB, in and out."""
    say(f"qk_norm_rope_rows {layout} far apart")
    T, D, stride = 130, 64, 20_000_000
    buf = torch.empty((T - 1) * stride + 20 * D, dtype=torch.bfloat16, device="cuda")
    at = lambda i, n: buf.as_strided((T, n, D), (stride, D, 1), i * D)  # noqa: E731
    q, k = at(0, 5), at(5, 2)
    q.copy_(randn(torch, 1, "bfloat16", T, 5, D))
    k.copy_(randn(torch, 2, "bfloat16", T, 2, D))
    f, w, lens = freqs(nxg, torch, D), randn(torch, 3, "float32", D), [100, 30]
    outs = at(7, 5), at(12, 2)
    nxg.qk_norm_rope_rows(q, k, w, w, f, offsets(lens), layout=layout, q_out=outs[0], k_out=outs[1])
    pos = places(torch, lens)
    for x, o in ((q, outs[0]), (k, outs[1])):
        check("y", o, *adapter_ref.qk_norm_rope(x.contiguous(), w, f, pos, layout, 1.0, 1e-6))
    dy = randn(torch, 4, "bfloat16", T, 5, D)
    grads = nxg.qk_norm_rope_rows_backward(dy, k, q, k, w, w, f, offsets(lens), layout=layout, dq=outs[0], dk=outs[1])
    for name, t, r in zip(("dq", "dw"), (grads[0], grads[2]), adapter_ref.qk_norm_rope_back(dy, q.contiguous(), w, f, pos, layout, 1.0, 1e-6)):
        check(name, t, *r)


# --- dropout -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,C", [(1, 1), (1, 8), (3, 7), (5, 64), (37, 1023), (33, 1024), (9, 2304), (700, 24), (5000, 2), (3, 8200), (2, 20001)])
def test_dropout(nxg, torch, dev, dtype, T, C):
    say(f"dropout_rows {dtype} T={T} C={C}")
    x, r = randn(torch, C, dtype, T, C), randn(torch, C + 1, dtype, T, C)
    for p, residual, seed, offset in ((0.1, r, 1234567890123, 7), (0.5, None, 2 ** 64 - 1, 2 ** 64 - 1)):
        y = nxg.dropout_rows(x, p, seed, offset, residual=residual)
        check("y", y, *adapter_ref.dropout(x, residual, p, seed, offset))


def test_dropout_probabilities(nxg, torch, dev):
    say("dropout_rows p")
    x = randn(torch, 1, "float32", 64, 256)
    assert torch.equal(nxg.dropout_rows(x, 0.0, 1), x)
    for p in (2.0 ** -16, 1 - 2.0 ** -16, 0.3, 1e-9):
        check(f"p={p}", nxg.dropout_rows(x, p, 5, 6), *adapter_ref.dropout(x, None, p, 5, 6))
    for p in (-0.1, 1.0, 1 - 1e-9, math.nan):
        with pytest.raises(ValueError, match="p="):
            nxg.dropout_rows(x, p, 1)
    for seed, offset in ((-1, 0), (1 << 64, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError, match="64-bit"):
            nxg.dropout_rows(x, 0.1, seed, offset)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_gradient_strides_and_in_place(nxg, torch, dev, dtype):
    """The same call without the residual on dy is the transposed map; strides and the type do not change the mask."""
    say(f"dropout_rows {dtype} gradient, strided, in place")
    T, C, p = 21, 200, 0.25                                       # 1 / (1 - p) is not exact, a product with 1 is
    keep = torch.from_numpy(adapter_ref.kept(T, C, p, 3, 4)).cuda()
    one = torch.ones(T, C, dtype=getattr(torch, dtype), device="cuda")
    dx = nxg.dropout_rows(one, p, 3, 4)
    assert torch.equal(dx != 0, keep) and float((dx[keep].double() - 4 / 3).abs().max()) <= 4 / 3 * (torch.finfo(dx.dtype).eps / 2 + 2.0 ** -23)
    for off in (0, 3):
        x = randn(torch, 3, dtype, T, C + 16)[:, off:off + C]
        r = randn(torch, 4, dtype, T, 2 * C)[:, :C]
        base = torch.full((T + 2, C + 16), 7.0, dtype=x.dtype, device="cuda")
        out = base[1:T + 1, off:off + C]
        ref = adapter_ref.dropout(x, r, p, 3, 4)
        check("y", nxg.dropout_rows(x, p, 3, 4, residual=r, out=out), *ref)
        assert (base[0] == 7).all() and (base[-1] == 7).all() and (base[:, off + C:] == 7).all() and (base[:, :off] == 7).all()
        a, b = x.clone(), r.clone()
        assert torch.equal(nxg.dropout_rows(a, p, 3, 4, residual=r, out=a), out)
        assert torch.equal(nxg.dropout_rows(x, p, 3, 4, residual=b, out=b), out)
        shared = r[:1].expand(T, C)                               # a residual row for all
        check("shared", nxg.dropout_rows(x, p, 3, 4, residual=shared), *adapter_ref.dropout(x, shared, p, 3, 4))


def test_dropout_special_values(nxg, torch, dev):
    """A dropped infinity or NaN leaves nothing; a kept one is one."""
    say("dropout_rows special values")
    x = randn(torch, 1, "bfloat16", 40, 64)
    x[3], x[5], x[7] = math.inf, math.nan, -math.inf
    check("y", nxg.dropout_rows(x, 0.5, 8, 9, residual=randn(torch, 2, "bfloat16", 40, 64)),
          *adapter_ref.dropout(x, randn(torch, 2, "bfloat16", 40, 64), 0.5, 8, 9))


def test_dropout_rows_far_apart(nxg, torch, dev):
    say("dropout_rows far apart")
    T, C, stride = 130, 1000, 20_000_000
    buf = torch.empty((T - 1) * stride + 3 * C, dtype=torch.bfloat16, device="cuda")
    x, r, out = (buf.as_strided((T, C), (stride, 1), i * C) for i in range(3))
    x.copy_(randn(torch, 3, "bfloat16", T, C))
    r.copy_(randn(torch, 4, "bfloat16", T, C))
    check("y", nxg.dropout_rows(x, 0.1, 1, 2, residual=r, out=out), *adapter_ref.dropout(x.contiguous(), r.contiguous(), 0.1, 1, 2))
    assert nxg.dropout_rows(x[:0], 0.1, 1).shape == (0, C)


def test_dropout_step_in_a_graph(nxg, torch, dev):
    """Replays draw new masks by the step that they read."""
    say("dropout_rows captured with a step")
    x = randn(torch, 1, "bfloat16", 50, 256)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nxg.dropout_rows(x, 0.1, 11, 5, step=step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nxg.dropout_rows(x, 0.1, 11, 5, step=step)
    for n in (0, 1, 1, 2 ** 40, -5, -6):
        step.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        check(f"step {n}", out, *adapter_ref.dropout(x, None, 0.1, 11, (5 + n) % 2 ** 64))
        assert torch.equal(out, nxg.dropout_rows(x, 0.1, 11, (5 + n) % 2 ** 64))
