"""CPU tests of include/nxg_rows.h and rows.py: every refusal is made before any device work, with its
reason; workspace sizes; the host's rotary frequencies against their formulas."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

P16 = 1 << 20            # an aligned address that no call here dereferences


@pytest.fixture()
def L(nxg):
    return nxg.load_library()


def refused(nxg, L, rc, word):
    assert rc == nxg.NXG_EINVAL, rc
    assert word in L.nxg_last_error().decode(), L.nxg_last_error()


def params(nxg, **kw):
    d = dict(type=nxg.TYPE_BF16, n_head=4, n_kv_head=2, head_dim=64, T_q=10, T_k=12, n_seqs=2, cu_q=P16, cu_k=P16, left=-1, right=-1, scale=0.125)
    d.update(kw)
    return nxg.rows._AttentionParams(*(d[f] for f, _ in nxg.rows._AttentionParams._fields_))


def rows(nxg, data=P16, ts=256, hs=64):
    return nxg.rows._Rows(data, ts, hs)


def forward(nxg, L, p=None, q=None, k=None, v=None, out=None, lse=P16, ws=None, ws_bytes=0):
    r = lambda x, **kw: ctypes.byref(x if x is not None else rows(nxg, **kw))  # noqa: E731
    return L.nxg_attention_rows(ctypes.byref(p or params(nxg)), r(q), r(k), r(v), r(out), lse, ws, ws_bytes, None)


BAD_PARAMS = [({"type": 0}, "type 0"), ({"type": 8}, "type 8"), ({"head_dim": 0}, "head_dim"), ({"head_dim": 60}, "head_dim=60"),
              ({"head_dim": 136}, "head_dim=136"), ({"n_head": 0}, "n_head"), ({"n_kv_head": 3}, "n_kv_head=3"), ({"n_kv_head": 0}, "n_kv_head"),
              ({"T_q": -1}, "T_q=-1"), ({"T_k": -1}, "T_k=-1"), ({"n_seqs": -1}, "n_seqs"), ({"left": -2}, "left=-2"), ({"right": -7}, "right=-7"),
              ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": math.inf}, "scale"), ({"scale": math.nan}, "scale"),
              ({"T_q": 1 << 30, "n_head": 4}, "too large"), ({"T_q": (1 << 30) + 1}, "T_q"), ({"cu_q": None}, "null"), ({"cu_k": None}, "null")]


@pytest.mark.parametrize("change,word", BAD_PARAMS, ids=str)
def test_attention_params_refused(nxg, L, change, word):
    refused(nxg, L, forward(nxg, L, params(nxg, **change)), word)
    if word != "null":
        p = ctypes.byref(params(nxg, **change))
        for f in (L.nxg_attention_rows_workspace_bytes, L.nxg_attention_rows_backward_workspace_bytes):
            assert f(p) == -nxg.NXG_EINVAL


BAD_ROWS = [({"data": None}, "null"), ({"data": P16 + 8}, "aligned"), ({"ts": 252}, "strides"), ({"hs": 66}, "strides"), ({"ts": -256}, "strides"),
            ({"hs": -64}, "strides"), ({"ts": 1 << 62}, "strides")]


@pytest.mark.parametrize("change,word", BAD_ROWS, ids=str)
@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_attention_rows_refused(nxg, L, name, change, word):
    refused(nxg, L, forward(nxg, L, **{name: rows(nxg, **change)}), word)
    assert f"{name} " in L.nxg_last_error().decode()


def test_overlapping_outputs_refused(nxg, L):
    for ts, hs in ((256, 56), (192, 64), (64, 256), (0, 64), (256, 0), (64, 576)):
        refused(nxg, L, forward(nxg, L, out=rows(nxg, ts=ts, hs=hs)), "overlap")
    assert forward(nxg, L, params(nxg, T_q=0), out=rows(nxg, ts=0)) == nxg.NXG_OK       # no rows: nothing to do
    assert forward(nxg, L, params(nxg, n_seqs=0)) == nxg.NXG_OK


def test_attention_workspace_refused(nxg, L):
    refused(nxg, L, forward(nxg, L, ws=None, ws_bytes=64), "workspace")
    refused(nxg, L, forward(nxg, L, ws=P16 + 4, ws_bytes=64), "workspace")
    refused(nxg, L, forward(nxg, L, ws=P16, ws_bytes=-1), "workspace")
    refused(nxg, L, forward(nxg, L, lse=None), "lse")
    refused(nxg, L, L.nxg_attention_rows(None, None, None, None, None, None, None, 0, None), "null")
    # one query over many keys shares them out; a long prompt does not
    few = ctypes.byref(params(nxg, T_q=1, T_k=65536, n_seqs=1))
    assert L.nxg_attention_rows_workspace_bytes(few) > 0
    assert L.nxg_attention_rows_workspace_bytes(ctypes.byref(params(nxg, T_q=65536, T_k=65536, n_seqs=1))) == 0


def test_attention_backward_refused(nxg, L):
    p = params(nxg)
    need = L.nxg_attention_rows_backward_workspace_bytes(ctypes.byref(p))
    assert need >= 2 * 4 * 10 * 4
    names = ["dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"]

    def call(ws=P16, n=need, **change):
        args = []
        for name in names:
            if name == "lse":
                args.append(change.get("lse", P16))
            else:
                args.append(ctypes.byref(change.get(name, rows(nxg))))
        return L.nxg_attention_rows_backward(ctypes.byref(p), *args, ws, n, None)
    for name in names:
        if name != "lse":
            refused(nxg, L, call(**{name: rows(nxg, data=P16 + 2)}), f"{name} must be 16-byte")
    for name in ("dq", "dk", "dv"):
        refused(nxg, L, call(**{name: rows(nxg, ts=0)}), "overlap")
    refused(nxg, L, call(lse=None), "lse")
    refused(nxg, L, call(ws=None), "workspace")
    refused(nxg, L, call(n=need - 1), "workspace")
    refused(nxg, L, call(ws=P16 + 8), "workspace")


def test_rope_refused(nxg, L):
    def call(type=nxg.TYPE_F32, x=None, T=4, H=2, D=64, freq=P16, n=64, layout=0, pos=None, cu=P16, n_seqs=1, out=None):
        x, out = (r if r is not None else rows(nxg, ts=128) for r in (x, out))
        return L.nxg_rope_rows(type, ctypes.byref(x), T, H, D, freq, n, layout, 1.0, 0, pos, cu, n_seqs, ctypes.byref(out), None)
    refused(nxg, L, call(type=8), "type 8")
    for kw in ({"T": -1}, {"H": 0}, {"D": 1}, {"D": 1025}):
        refused(nxg, L, call(**kw), "T=")
    for n in (0, 1, 63, 66, -2):
        refused(nxg, L, call(n=n), "n_rot")
    refused(nxg, L, call(layout=2), "layout")
    refused(nxg, L, call(freq=None), "null")
    refused(nxg, L, call(cu=None), "null")
    refused(nxg, L, call(n_seqs=0), "n_seqs")
    refused(nxg, L, call(x=rows(nxg, data=None)), "null")
    refused(nxg, L, call(x=rows(nxg, data=P16 + 2)), "aligned")
    refused(nxg, L, call(x=rows(nxg, ts=-128)), "strides")
    refused(nxg, L, call(out=rows(nxg, data=P16 * 2, ts=100)), "overlap")
    refused(nxg, L, call(out=rows(nxg, ts=256)), "other strides")
    assert call(T=0) == nxg.NXG_OK


def test_layer_norm_refused(nxg, L):
    def fwd(type=nxg.TYPE_BF16, x=P16, xs=64, w=P16, b=P16, wt=nxg.TYPE_F32, eps=1e-5, T=4, C=64, y=P16, ys=64):
        return L.nxg_layer_norm_rows(type, x, xs, w, b, wt, eps, T, C, y, ys, None, None, None)
    refused(nxg, L, fwd(type=2), "type 2")
    refused(nxg, L, fwd(wt=nxg.TYPE_F16), "weight type")
    for kw in ({"T": -1}, {"C": 0}):
        refused(nxg, L, fwd(**kw), "T=")
    for eps in (-1.0, math.nan, math.inf):
        refused(nxg, L, fwd(eps=eps), "eps")
    refused(nxg, L, fwd(x=None), "x is null")
    refused(nxg, L, fwd(y=P16 + 1), "y is null or not aligned")
    refused(nxg, L, fwd(xs=-1), "stride")
    refused(nxg, L, fwd(ys=63), "stride 63 of y")
    refused(nxg, L, fwd(w=P16 + 2), "w or b")
    assert fwd(T=0) == nxg.NXG_OK
    need = L.nxg_layer_norm_rows_workspace_bytes(4, 64)
    assert need > 0 and L.nxg_layer_norm_rows_workspace_bytes(-1, 64) == -nxg.NXG_EINVAL

    def back(type=nxg.TYPE_BF16, dy=P16, x=P16, mean=P16, rstd=P16, w=P16, wt=nxg.TYPE_F32, T=4, C=64, dx=P16, dxs=64, dw=P16, db=P16, ws=P16, n=need):
        return L.nxg_layer_norm_rows_backward(type, dy, 64, x, 64, mean, rstd, w, wt, T, C, dx, dxs, dw, db, ws, n, None)
    refused(nxg, L, back(type=9), "type 9")
    refused(nxg, L, back(wt=nxg.TYPE_F16), "weight type")
    refused(nxg, L, back(dy=None), "dy is null")
    refused(nxg, L, back(x=P16 + 1), "x is null or not aligned")
    refused(nxg, L, back(mean=None), "mean")
    refused(nxg, L, back(dxs=60), "stride 60 of dx")
    refused(nxg, L, back(dw=P16 + 2), "aligned")
    refused(nxg, L, back(ws=None), "workspace")
    refused(nxg, L, back(n=need - 1), "workspace")
    assert back(dx=None, dw=None, db=None, ws=None, n=0) == nxg.NXG_OK
    assert back(T=0, dw=None, db=None, ws=None, n=0) == nxg.NXG_OK


def test_rope_frequencies(nxg):
    for n, base in ((64, 1e4), (32, 1e5), (2, 500.0), (128, 1e6)):
        f, m = nxg.rope_frequencies(n, base)
        want = base ** (-2.0 * np.arange(n // 2) / n)
        assert m == 1.0 and np.allclose(f, want, rtol=1e-14, atol=0)
        assert np.allclose(nxg.rope_frequencies(n, base, "linear", 4.0)[0], want / 4, rtol=1e-14, atol=0)
    # ntk: as the encoder scales its base past the trained length, so the slowest pair turns 1 / factor as fast
    f, m = nxg.rope_frequencies(64, 1e5, "ntk", 8.0)
    assert m == 1.0 and f[0] == 1.0 and math.isclose(f[-1], nxg.rope_frequencies(64, 1e5)[0][-1] / 8, rel_tol=1e-13)
    # by_parts: pairs of 32 turns over the trained length as they are, of one turn or less by the factor
    f, m = nxg.rope_frequencies(64, 1e4, "by_parts", 16.0, 4096)
    plain = nxg.rope_frequencies(64, 1e4)[0]
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(m, 0.1 * math.log(16) + 1, rel_tol=1e-7)
    assert np.array_equal(f[turns >= 32], plain[turns >= 32]) and np.allclose(f[turns <= 1], plain[turns <= 1] / 16, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    g = (turns[mid] - 1) / 31
    assert mid.any() and np.allclose(f[mid], plain[mid] * ((1 - g) / 16 + g), rtol=1e-13, atol=0)
    for args in ((0, 1e4), (63, 1e4), (-4, 1e4), (64, 0.0), (64, -1.0), (64, math.inf), (64, 1e4, "linear", 0.5), (64, 1e4, "ntk", math.nan),
                 (2, 1e4, "ntk", 2.0), (64, 1e4, "by_parts", 2.0, 0), (64, 1e4, "cubic")):
        with pytest.raises(ValueError):
            nxg.rope_frequencies(*args)


def test_host_tensors_refused(nxg):
    """No CPU fallback: tensors that are not on the current device raise."""
    torch = pytest.importorskip("torch")
    x, q = torch.zeros(4, 8), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="current device"):
        nxg.layer_norm_rows(x)
    with pytest.raises(ValueError, match="current device"):
        nxg.rope_rows(q, torch.zeros(32, dtype=torch.float64), [0, 4])
    with pytest.raises(ValueError, match="current device"):
        nxg.attention_rows(q, q, q, [0, 4])
    with pytest.raises(ValueError, match="does not take"):
        nxg.attention_rows(q.float(), q.float(), q.float(), [0, 4])
    with pytest.raises(ValueError, match="does not take"):
        nxg.layer_norm_rows(x.double())


def test_sizes_past_a_launch_refused(nxg, L):
    """More workgroups than a launch has: said before any device work."""
    for kw in ({"T_q": 1 << 30, "n_head": 1, "n_kv_head": 1, "T_k": 1 << 30}, {"n_seqs": 1 << 24}, {"T_k": 1 << 29, "n_kv_head": 4}):
        refused(nxg, L, forward(nxg, L, params(nxg, **kw)), "too large")
    x, n = ctypes.byref(rows(nxg, ts=64)), 1 << 25
    refused(nxg, L, L.nxg_rope_rows(nxg.TYPE_F32, x, n, 100, 64, P16, 64, 0, 1.0, 0, None, P16, 1, ctypes.byref(rows(nxg, data=2 * P16, ts=6400)), None), "too large")
    for T, C in ((1 << 24, 1025), (1 << 26, 1024), (4, (1 << 23) + 1)):
        refused(nxg, L, L.nxg_layer_norm_rows(nxg.TYPE_F32, P16, C, None, None, nxg.TYPE_F32, 1e-5, T, C, P16, C, None, None, None), "too large")
        assert L.nxg_layer_norm_rows_workspace_bytes(T, C) == -nxg.NXG_EINVAL


def test_layer_norm_in_place_with_another_stride_refused(nxg, L):
    f32 = nxg.TYPE_F32
    refused(nxg, L, L.nxg_layer_norm_rows(f32, P16, 128, None, None, f32, 1e-5, 4, 64, P16, 64, None, None, None), "another stride")
    for dys, xs, dx in ((128, 64, P16), (64, 128, 2 * P16)):
        refused(nxg, L, L.nxg_layer_norm_rows_backward(f32, P16, dys, 2 * P16, xs, P16, P16, None, f32, 4, 64, dx, 64, None, None, None, 0, None),
                "another stride")


def test_outputs_over_other_tensors_refused(nxg, L):
    p = params(nxg, T_q=12)
    for name in ("q", "k", "v"):
        at = {n: rows(nxg, data=(2 + i) * P16) for i, n in enumerate(("q", "k", "v"))}
        at["out"] = rows(nxg, data=at[name].data)
        refused(nxg, L, forward(nxg, L, p, **at), "out is another tensor")
    names = ["dout", "q", "k", "v", "out", "dq", "dk", "dv"]
    need = L.nxg_attention_rows_backward_workspace_bytes(ctypes.byref(p))
    for i, name in enumerate(names[5:], 5):
        for other in names[:i]:
            at = {n: rows(nxg, data=(2 + k) * P16) for k, n in enumerate(names)}
            at[name] = rows(nxg, data=at[other].data)
            a = [ctypes.byref(at[n]) for n in names]
            refused(nxg, L, L.nxg_attention_rows_backward(ctypes.byref(p), *a[:5], P16, *a[5:], P16, need, None), f"{name} is another tensor")
