"""GPU: rope_rows, layer_norm_rows and layer_norm_rows_backward against 64 bits (rows_ref.py, with the
bounds of their roundings)."""
from __future__ import annotations

import math

import numpy as np
import pytest

import rows_ref

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


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


def positions_of(lens):
    return np.concatenate([np.arange(n) for n in lens] or [np.zeros(0)]).astype(np.int64)


# --- rotary positions ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,n", [(64, 64), (64, 32), (128, 128), (80, 40), (6, 2), (63, 20), (256, 256)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rope(nxg, torch, dev, dtype, layout, D, n, inverse):
    say(f"rope_rows {dtype} {layout} D={D} n={n} inverse={inverse}")
    lens = [1, 40, 3, 77]
    x = randn(torch, D, dtype, sum(lens), 5, D)
    f, m = nxg.rope_frequencies(n, 10000.0)
    assert m == 1.0
    f = torch.from_numpy(f).cuda()
    y = nxg.rope_rows(x, f, np.concatenate([[0], np.cumsum(lens)]), layout=layout, inverse=inverse, mscale=1.25)
    ref = rows_ref.rope(x, f, torch.from_numpy(positions_of(lens)).cuda(), layout, 1.25, inverse)
    rows_ref.check("rope", y, *ref)


@pytest.mark.parametrize("scaling,factor,train_len", [("none", 1.0, 0), ("linear", 4.0, 0), ("ntk", 8.0, 0), ("by_parts", 16.0, 4096)])
def test_rope_far_positions(nxg, torch, dev, scaling, factor, train_len):
    """Positions up to the ends of int32, negative ones too: the angle keeps its place in the turn."""
    say(f"rope_rows far positions {scaling}")
    pos = torch.tensor([0, 1, -1, 65535, 1000003, 2 ** 31 - 1, -2 ** 31, 123456789], dtype=torch.int32, device="cuda")
    x = randn(torch, 1, "float32", len(pos), 3, 64)
    f, m = nxg.rope_frequencies(64, 100000.0, scaling, factor, train_len)
    f = torch.from_numpy(f).cuda()
    y = nxg.rope_rows(x, f, positions=pos, mscale=m)
    rows_ref.check("rope", y, *rows_ref.rope(x, f, pos.long(), "half", m, False))


def test_rope_gradient_is_the_inverse(nxg, torch, dev):
    """<dy, rope(x)> = <rope_inverse(dy), x>: the inverse call is the transposed map, so the gradient."""
    say("rope_rows inverse is the transpose")
    x, dy = randn(torch, 1, "float32", 50, 4, 64), randn(torch, 2, "float32", 50, 4, 64)
    f, m = nxg.rope_frequencies(32, 10000.0, "by_parts", 4.0, 16)
    f = torch.from_numpy(f).cuda()
    a = (dy.double() * nxg.rope_rows(x, f, [0, 20, 50], mscale=m).double()).sum()
    b = (nxg.rope_rows(dy, f, [0, 20, 50], mscale=m, inverse=True).double() * x.double()).sum()
    assert abs(float(a - b)) <= 2 * m * (2.0 ** -20) * float((dy.double().abs().sum(2) * x.double().abs().sum(2)).sum())


def test_rope_turns_as_qk_prep_does(nxg, torch, dev):
    """inverse=True is the sense of the encoder's nxg_qk_prep (its DyT taken out: tanh(a x) / a to x)."""
    say("rope_rows against qk_prep")
    x = randn(torch, 3, "float32", 30, 2, 64)
    cos, sin = nxg.rope_table(30, 10000.0)
    a = torch.full((64,), 1e-3, device="cuda")
    y = nxg.qk_prep(x.reshape(30, 128), a, 1 / a, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), [0, 30], 2).reshape(30, 2, 64)
    f = torch.from_numpy(nxg.rope_frequencies(64, 10000.0)[0]).cuda()
    z = nxg.rope_rows(x, f, [0, 30], inverse=True)
    # tanh(t) / t = 1 - t^2 / 3 ..., t = 1e-3 |x| at most 5e-3: 1e-5 of a value; the table's fp32 angles: 30 2^-24
    assert float((y - z).abs().max()) <= 2 * float(x.abs().max()) * (1e-5 + 30 * 2.0 ** -23)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_in_place_and_strides(nxg, torch, dev, dtype, layout):
    say(f"rope_rows {dtype} {layout} in place, strided")
    lens = [30, 11]
    T, D = sum(lens), 64
    cu = np.concatenate([[0], np.cumsum(lens)])
    f = torch.from_numpy(nxg.rope_frequencies(32, 10000.0)[0]).cuda()
    rows = randn(torch, 4, dtype, T, 9, D)
    before = rows.clone()
    ref = rows_ref.rope(before[:, 1:6], f, torch.from_numpy(positions_of(lens)).cuda(), layout, 1.0, False)
    part = rows[:, 1:6]
    out = nxg.rope_rows(part, f, cu, layout=layout, out=part)
    assert out.data_ptr() == part.data_ptr()
    rows_ref.check("in place", out, *ref)
    assert torch.equal(rows[:, 0], before[:, 0]) and torch.equal(rows[:, 6:], before[:, 6:])
    # rows that are not 16-byte aligned, and head-major ones
    odd = randn(torch, 4, dtype, T, 9, D + 1)[:, 1:6, 1:]
    odd.copy_(before[:, 1:6])
    rows_ref.check("odd", nxg.rope_rows(odd, f, cu, layout=layout), *ref)
    heads = before[:, 1:6].transpose(0, 1).contiguous().transpose(0, 1)
    to = torch.empty(5, T, D, dtype=rows.dtype, device="cuda").transpose(0, 1)
    rows_ref.check("head-major", nxg.rope_rows(heads, f, cu, layout=layout, out=to), *ref)


def test_rope_sizes(nxg, torch, dev):
    say("rope_rows one token, many heads, many documents")
    f = torch.from_numpy(nxg.rope_frequencies(64, 10000.0)[0]).cuda()
    for T, H, lens in ((1, 1, [1]), (1, 300, [1]), (2000, 3, [1] * 1500 + [0, 500]), (5000, 24, [5000])):
        x = randn(torch, T, "bfloat16", T, H, 64)
        y = nxg.rope_rows(x, f, np.concatenate([[0], np.cumsum(lens)]))
        rows_ref.check(f"{T}", y, *rows_ref.rope(x, f, torch.from_numpy(positions_of(lens)).cuda(), "half", 1.0, False))
    assert nxg.rope_rows(x[:0], f, [0, 0]).shape == (0, 24, 64)


# --- layer norm ------------------------------------------------------------------------------------

COLS = [1, 2, 7, 64, 100, 1023, 1024, 2304, 4096, 8192, 8200, 10001]


@pytest.mark.parametrize("dtype,wtype", [("float32", "float32"), ("float16", "float32"), ("float16", "float16"),
                                         ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("C", COLS)
def test_layer_norm(nxg, torch, dev, dtype, wtype, C):
    say(f"layer_norm_rows {dtype} {wtype} C={C}")
    T, eps = 37, 1e-5
    x = randn(torch, C, dtype, T, C) * 2 + 1
    w, b, dy = randn(torch, C + 1, wtype, C), randn(torch, C + 2, wtype, C), randn(torch, C + 3, dtype, T, C)
    y, mean, rstd = nxg.layer_norm_rows(x, w, b, eps)
    for name, t, ref in zip(("y", "mean", "rstd"), (y, mean, rstd), rows_ref.layer_norm(x, w, b, eps)):
        rows_ref.check(name, t, *ref)
    for name, t, ref in zip(("dx", "dw", "db"), nxg.layer_norm_rows_backward(dy, x, mean, rstd, w), rows_ref.layer_norm_back(dy, x, mean, rstd, w)):
        rows_ref.check(name, t, *ref)


@pytest.mark.parametrize("T", [0, 1, 2, 5, 511, 2049, 9000])
@pytest.mark.parametrize("C", [64, 1024, 2600])
def test_layer_norm_rows_counts(nxg, torch, dev, T, C):
    say(f"layer_norm_rows T={T} C={C}")
    x, dy = randn(torch, T, "bfloat16", T, C), randn(torch, T + 1, "bfloat16", T, C)
    y, mean, rstd = nxg.layer_norm_rows(x, None, None, 1e-5)
    grads = nxg.layer_norm_rows_backward(dy, x, mean, rstd)
    if T == 0:
        assert (grads[1] == 0).all() and (grads[2] == 0).all() and y.shape == (0, C)
        return
    rows_ref.check("y", y, *rows_ref.layer_norm(x, None, None, 1e-5)[0])
    for name, t, ref in zip(("dx", "dw", "db"), grads, rows_ref.layer_norm_back(dy, x, mean, rstd, None)):
        rows_ref.check(name, t, *ref)
    again = nxg.layer_norm_rows_backward(dy, x, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("C", [1024, 1000, 9000])
def test_layer_norm_strides_and_in_place(nxg, torch, dev, C):
    say(f"layer_norm_rows strided C={C}")
    T = 21
    w, b = randn(torch, 1, "float32", C), randn(torch, 2, "float32", C)
    for off in (0, 3):                                # 3: rows off 16 bytes
        x = randn(torch, 3, "bfloat16", T, C + 16)[:, off:off + C]
        dy = randn(torch, 4, "bfloat16", T, 2 * C)[:, :C]
        base = torch.full((T + 2, C + 16), 7.0, dtype=torch.bfloat16, device="cuda")
        out = base[1:T + 1, off:off + C]
        y, mean, rstd = nxg.layer_norm_rows(x, w, b, 1e-5, out=out)
        rows_ref.check("y", y, *rows_ref.layer_norm(x, w, b, 1e-5)[0])
        ref = rows_ref.layer_norm_back(dy, x, mean, rstd, w)
        dx, dw, db = nxg.layer_norm_rows_backward(dy, x, mean, rstd, w, dx=out)
        for name, t, r in zip(("dx", "dw", "db"), (dx, dw, db), ref):
            rows_ref.check(name, t, *r)
        assert (base[0] == 7).all() and (base[-1] == 7).all() and (base[:, off + C:] == 7).all() and (base[:, :off] == 7).all()
        dz = dy.clone()
        assert torch.equal(nxg.layer_norm_rows_backward(dz, x, mean, rstd, w, dx=dz)[0], dx)
        xc = x.clone()
        assert torch.equal(nxg.layer_norm_rows(xc, w, b, 1e-5, out=xc)[0], nxg.layer_norm_rows(x, w, b, 1e-5)[0])


def test_layer_norm_special_rows(nxg, torch, dev):
    """Constant rows (variance 0), huge and tiny ones, a row with an infinity or a NaN: others do not
    change."""
    say("layer_norm_rows special rows")
    x = randn(torch, 1, "float32", 8, 256)
    x[1] = 3.0
    x[2] *= 1e15
    x[3] *= 1e-15
    plain = nxg.layer_norm_rows(x)[0]
    rows_ref.check("y", plain, *rows_ref.layer_norm(x, None, None, 1e-5)[0])
    z = x.clone()
    z[5, 7], z[6, 0] = math.inf, math.nan
    y = nxg.layer_norm_rows(z)[0]
    keep = [0, 1, 2, 3, 4, 7]
    assert torch.equal(y[keep], plain[keep]) and torch.isnan(y[6]).all() and torch.isnan(y[5]).any()


def test_layer_norm_gradient_against_differences(nxg, torch, dev):
    say("layer_norm_rows gradient against differences")
    T, C = 6, 96
    x, w, b, dy = randn(torch, 1, "float32", T, C), randn(torch, 2, "float32", C), randn(torch, 3, "float32", C), randn(torch, 4, "float32", T, C)
    _, mean, rstd = nxg.layer_norm_rows(x, w, b)
    grads = nxg.layer_norm_rows_backward(dy, x, mean, rstd, w)
    f = lambda *a: float((rows_ref.layer_norm(*a, 1e-5)[0][0] * dy.double()).sum())  # noqa: E731
    args = [x.double(), w.double(), b.double()]
    for i, grad in enumerate(grads):
        step = torch.sign(randn(torch, 9 + i, "float32", *args[i].shape)).double() * 2.0 ** -16
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step, args[i] - step
        diff = (f(*up) - f(*down)) / 2
        want = float((grad.double() * step).sum())
        # fp32 roundings of the gradient (2^-18 of its size is far above them) and the third-order term
        assert abs(diff - want) <= 2.0 ** -18 * float((grad.double().abs() * step.abs()).sum()) + 2.0 ** -36, (i, diff, want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_rows_far_apart(nxg, torch, dev, layout):
    """Rows over more than 4 GiB, in and out."""
    say(f"rope_rows {layout} far apart")
    T, H, D, stride = 130, 5, 64, 20_000_000
    buf = torch.empty((T - 1) * stride + 2 * H * D, dtype=torch.bfloat16, device="cuda")
    x, out = (buf.as_strided((T, H, D), (stride, D, 1), i * H * D) for i in range(2))
    x.copy_(randn(torch, 1, "bfloat16", T, H, D))
    f = torch.from_numpy(nxg.rope_frequencies(D, 10000.0)[0]).cuda()
    nxg.rope_rows(x, f, [0, 100, T], layout=layout, out=out)
    rows_ref.check("y", out, *rows_ref.rope(x.contiguous(), f, torch.from_numpy(positions_of([100, 30])).cuda(), layout, 1.0, False))


@pytest.mark.parametrize("C", [1024, 1000, 9000])
def test_layer_norm_rows_far_apart(nxg, torch, dev, C):
    say(f"layer_norm_rows far apart C={C}")
    T, stride = 130, 20_000_000
    buf = torch.empty((T - 1) * stride + 3 * C, dtype=torch.bfloat16, device="cuda")
    x, dy, out = (buf.as_strided((T, C), (stride, 1), i * C) for i in range(3))
    x.copy_(randn(torch, 3, "bfloat16", T, C))
    dy.copy_(randn(torch, 4, "bfloat16", T, C))
    w, b = randn(torch, 1, "float32", C), randn(torch, 2, "float32", C)
    y, mean, rstd = nxg.layer_norm_rows(x, w, b, 1e-5, out=out)
    rows_ref.check("y", y, *rows_ref.layer_norm(x.contiguous(), w, b, 1e-5)[0])
    ref = rows_ref.layer_norm_back(dy.contiguous(), x.contiguous(), mean, rstd, w)
    for name, t, r in zip(("dx", "dw", "db"), nxg.layer_norm_rows_backward(dy, x, mean, rstd, w, dx=out), ref):
        rows_ref.check(name, t, *r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [64, 1000, 4096, 9000])
@pytest.mark.parametrize("into", ["dy", "x"])
def test_layer_norm_gradients_in_place(nxg, torch, dev, dtype, C, into):
    """dx over dy or over x: the weights' gradients are those of the rows as they were."""
    say(f"layer_norm_rows_backward {dtype} C={C} dx over {into}")
    T = 600
    x, dy, w = randn(torch, 1, dtype, T, C), randn(torch, 2, dtype, T, C), randn(torch, 3, "float32", C)
    _, mean, rstd = nxg.layer_norm_rows(x, w)
    want = nxg.layer_norm_rows_backward(dy, x, mean, rstd, w)
    got = nxg.layer_norm_rows_backward(dy, x, mean, rstd, w, dx=dy if into == "dy" else x)
    for name, a, b in zip(("dx", "dw", "db"), got, want):
        assert torch.equal(a, b), name
