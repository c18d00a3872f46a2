"""CPU tests of qk_norm_rope_rows, dropout_rows and adapter_rows (include/nxg_rows.h, rows.py): every refusal is made before any device
work, with its reason; workspace sizes."""
from __future__ import annotations

import ctypes
import math

import pytest

P16 = 1 << 20            # an aligned address that no call here dereferences


class QkNormRopeParams(ctypes.Structure):
    """struct nxg_qk_norm_rope_params."""
    _fields_ = [("type", ctypes.c_int32), ("T", ctypes.c_int32), ("n_head", ctypes.c_int32), ("n_kv_head", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("wq", ctypes.c_void_p), ("wk", ctypes.c_void_p), ("w_type", ctypes.c_int32),
                ("eps", ctypes.c_float), ("freq", ctypes.c_void_p), ("n_rot", ctypes.c_int32), ("layout", ctypes.c_int32),
                ("mscale", ctypes.c_float), ("positions", ctypes.c_void_p), ("cu", ctypes.c_void_p), ("n_seqs", ctypes.c_int32)]


class AdapterParams(ctypes.Structure):
    """struct nxg_adapter_rows_params."""
    _fields_ = [("type", ctypes.c_int32), ("w_type", ctypes.c_int32), ("T", ctypes.c_int32), ("n_in", ctypes.c_int32),
                ("n_out", ctypes.c_int32), ("rank", ctypes.c_int32), ("n_adapters", ctypes.c_int32), ("n_seqs", ctypes.c_int32),
                ("cu", ctypes.c_void_p), ("ids", ctypes.c_void_p), ("a", ctypes.c_void_p), ("b", ctypes.c_void_p),
                ("scale", ctypes.c_float)]


def test_words_of_the_params(nxg):
    assert nxg.rows._qk_params.size == ctypes.sizeof(QkNormRopeParams)
    assert nxg.rows._adapter_params.size == ctypes.sizeof(AdapterParams)
    q = QkNormRopeParams(*range(1, 9), 0.5, *range(10, 13), 0.25, *range(14, 17))
    assert bytes(q) == nxg.rows._qk_params.pack(*range(1, 9), 0.5, *range(10, 13), 0.25, *range(14, 17))
    a = AdapterParams(*range(1, 13), 0.5)
    assert bytes(a) == nxg.rows._adapter_params.pack(*range(1, 13), 0.5)


@pytest.fixture()
def L(nxg):
    return nxg.load_library()


def refused(nxg, L, rc, word):
    assert rc == nxg.NXG_EINVAL, rc
    assert word in L.nxg_last_error().decode(), L.nxg_last_error()


def struct(cls, **kw):
    return cls(*(kw[f] for f, _ in cls._fields_))


def rows(nxg, data=P16, ts=256, hs=64):
    return nxg.rows._Rows(data, ts, hs)


# --- norms of queries and keys ---------------------------------------------------------------------

def qk_params(nxg, **kw):
    d = dict(type=nxg.TYPE_BF16, T=10, n_head=4, n_kv_head=2, head_dim=64, wq=P16, wk=P16, w_type=nxg.TYPE_F32, eps=1e-6, freq=P16, n_rot=64,
             layout=0, mscale=1.0, positions=None, cu=P16, n_seqs=1)
    d.update(kw)
    return struct(QkNormRopeParams, **d)


def qk(nxg, L, p=None, **kw):
    at = {n: rows(nxg, data=(i + 2) * P16) for i, n in enumerate(("q", "k", "q_out", "k_out"))}
    at.update(kw)
    return L.nxg_qk_norm_rope_rows(ctypes.byref(p or qk_params(nxg)), *(None if at[n] is None else ctypes.byref(at[n]) for n in ("q", "k", "q_out", "k_out")), None)


NEED = 768 * 64 * 4


def qk_back(nxg, L, p=None, dwq=P16, dwk=P16, ws=P16, n=NEED, **kw):
    names = ("dq_out", "dk_out", "q", "k", "dq", "dk")
    at = {m: rows(nxg, data=(i + 2) * P16) for i, m in enumerate(names)}
    at.update(kw)
    return L.nxg_qk_norm_rope_rows_backward(ctypes.byref(p or qk_params(nxg)), *(None if at[m] is None else ctypes.byref(at[m]) for m in names), dwq, dwk, ws, n, None)


BAD_QK = [({"type": 2}, "type 2"), ({"w_type": 1}, "weight type 1"), ({"T": -1}, "T=-1"), ({"n_head": 0}, "n_head=0"), ({"n_kv_head": -1}, "n_kv_head=-1"),
          ({"head_dim": 1}, "head_dim=1"), ({"head_dim": 1025}, "head_dim"), ({"n_head": 65537}, "n_head"), ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"),
          ({"n_rot": 0}, "n_rot=0"), ({"n_rot": 63}, "n_rot=63"), ({"n_rot": 66}, "n_rot=66"), ({"layout": 2}, "layout 2")]


@pytest.mark.parametrize("change,word", BAD_QK, ids=str)
def test_qk_params_refused(nxg, L, change, word):
    p = qk_params(nxg, **change)
    refused(nxg, L, qk(nxg, L, p), word)
    refused(nxg, L, qk_back(nxg, L, p), word)
    assert L.nxg_qk_norm_rope_rows_workspace_bytes(ctypes.byref(p)) == -nxg.NXG_EINVAL


def test_qk_arrays_refused(nxg, L):
    for change, word in (({"freq": None}, "null freq"), ({"cu": None}, "null freq"), ({"n_seqs": 0}, "n_seqs"), ({"wq": None}, "wq"), ({"wk": None}, "wk"),
                         ({"wk": P16 + 2}, "wk")):
        refused(nxg, L, qk(nxg, L, qk_params(nxg, **change)), word)
        refused(nxg, L, qk_back(nxg, L, qk_params(nxg, **change)), word)
    for name in ("q", "k", "q_out", "k_out"):
        for bad, word in ((None, "null"), (rows(nxg, data=None), "null"), (rows(nxg, data=P16 + 1), "aligned"), (rows(nxg, ts=-256), "strides"), (rows(nxg, hs=1 << 62), "strides")):
            refused(nxg, L, qk(nxg, L, **{name: bad}), word)
            assert f"{name} " in L.nxg_last_error().decode()
    for name in ("q_out", "k_out"):
        for ts, hs in ((256, 56), (192 if name == "q_out" else 64, 64), (0, 64), (256, 0)):
            refused(nxg, L, qk(nxg, L, **{name: rows(nxg, data=9 * P16, ts=ts, hs=hs)}), "overlap")
    refused(nxg, L, qk(nxg, L, q_out=rows(nxg, data=2 * P16, ts=512)), "other strides")
    for kw in ({"q_out": rows(nxg, data=3 * P16)}, {"k_out": rows(nxg, data=2 * P16)}, {"q_out": rows(nxg, data=5 * P16)}):
        refused(nxg, L, qk(nxg, L, **kw), "another tensor")
    refused(nxg, L, qk(nxg, L, qk_params(nxg, T=1 << 30, n_head=400, n_kv_head=0, head_dim=1024), q=rows(nxg, ts=409600, hs=1024),
                       q_out=rows(nxg, data=2 * P16, ts=409600, hs=1024)), "too large")
    assert qk(nxg, L, qk_params(nxg, T=0)) == nxg.NXG_OK
    refused(nxg, L, L.nxg_qk_norm_rope_rows(None, None, None, None, None, None), "null params")


def test_qk_backward_refused(nxg, L):
    assert L.nxg_qk_norm_rope_rows_workspace_bytes(ctypes.byref(qk_params(nxg))) == NEED
    for kw in ({"ws": None}, {"ws": P16 + 8}, {"n": NEED - 1}):
        refused(nxg, L, qk_back(nxg, L, **kw), "workspace")
    for kw in ({"dwq": None}, {"dwk": None}, {"dwq": P16 + 2}):
        refused(nxg, L, qk_back(nxg, L, **kw), "dwq or dwk")
    for name in ("dq_out", "dk_out", "q", "k", "dq", "dk"):
        refused(nxg, L, qk_back(nxg, L, **{name: rows(nxg, data=P16 + 1)}), "aligned")
    for name in ("dq", "dk"):
        refused(nxg, L, qk_back(nxg, L, **{name: rows(nxg, data=9 * P16, ts=64)}), "overlap")
        for other in ("q", "k", "dq_out", "dk_out"):
            at = {other: rows(nxg, data=9 * P16), name: rows(nxg, data=9 * P16)}
            if name[1] == other[0] or other.startswith(name):
                at[name] = rows(nxg, data=9 * P16, ts=512)
                refused(nxg, L, qk_back(nxg, L, **at), "other strides")
            else:
                refused(nxg, L, qk_back(nxg, L, **at), "another tensor")
    refused(nxg, L, qk_back(nxg, L, dq=rows(nxg, data=9 * P16), dk=rows(nxg, data=9 * P16)), "another tensor")


# --- dropout ---------------------------------------------------------------------------------------

def test_dropout_refused(nxg, L):
    def call(type=nxg.TYPE_F32, x=P16, xs=64, r=2 * P16, rs=64, T=4, C=64, p=0.1, step=None, out=3 * P16, os=64):
        return L.nxg_dropout_rows(type, x, xs, r, rs, T, C, p, 1, 2, step, out, os, None)
    refused(nxg, L, call(type=8), "type 8")
    for kw in ({"T": -1}, {"C": 0}, {"C": (1 << 30) + 1}):
        refused(nxg, L, call(**kw), "T=")
    for p in (-0.1, 1.0, 2.0, 1 - 2.0 ** -18, math.nan, math.inf):
        refused(nxg, L, call(p=p), "p=")
    refused(nxg, L, call(x=None), "x is null")
    refused(nxg, L, call(r=P16 + 2), "residual is null or not aligned")
    refused(nxg, L, call(out=None), "out is null")
    refused(nxg, L, call(xs=-1), "stride -1 of x")
    refused(nxg, L, call(os=63), "stride 63 of out")
    refused(nxg, L, call(step=P16 + 4), "step")
    refused(nxg, L, call(out=P16, xs=128), "another stride")
    refused(nxg, L, call(out=2 * P16, rs=128), "another stride")
    refused(nxg, L, call(T=1 << 30, C=1 << 20, xs=1 << 20, rs=1 << 20, os=1 << 20), "too large")
    assert call(T=0) == nxg.NXG_OK


# --- low-rank adapters -----------------------------------------------------------------------------

def adapter_params(nxg, **kw):
    d = dict(type=nxg.TYPE_BF16, w_type=nxg.TYPE_BF16, T=10, n_in=64, n_out=128, rank=16, n_adapters=3, n_seqs=2, cu=P16, ids=P16, a=P16, b=2 * P16, scale=1.0)
    d.update(kw)
    return struct(AdapterParams, **d)


def adapter(nxg, L, p=None, x=3 * P16, xs=64, base=4 * P16, bs=128, y=5 * P16, ys=128, s=6 * P16):
    return L.nxg_adapter_rows(ctypes.byref(p or adapter_params(nxg)), x, xs, base, bs, y, ys, s, None)


def adapter_back(nxg, L, p=None, dy=3 * P16, dys=128, x=4 * P16, xs=64, s=5 * P16, base=6 * P16, bs=64, dx=7 * P16, dxs=64, da=8 * P16, db=9 * P16, ws=10 * P16, n=None):
    p = p or adapter_params(nxg)
    n = L.nxg_adapter_rows_backward_workspace_bytes(ctypes.byref(p)) if n is None else n
    return L.nxg_adapter_rows_backward(ctypes.byref(p), dy, dys, x, xs, s, base, bs, dx, dxs, da, db, ws, n, None)


BAD_ADAPTERS = [({"type": 2}, "type 2"), ({"w_type": 0}, "weight type 0"), ({"w_type": 1}, "weight type 1"), ({"type": 0, "w_type": 2}, "weight type 2"),
                ({"T": -1}, "T=-1"), ({"T": 1 << 24}, "T="), ({"n_seqs": -1}, "n_seqs"), ({"n_seqs": 1 << 22}, "n_seqs"), ({"n_in": 0}, "n_in=0"),
                ({"n_out": (1 << 20) + 1}, "n_out"), ({"rank": 0}, "rank=0"), ({"rank": 129}, "rank=129"), ({"n_adapters": 0}, "n_adapters=0"),
                ({"n_adapters": 1 << 22}, "too large"), ({"scale": math.inf}, "scale"), ({"scale": math.nan}, "scale")]


@pytest.mark.parametrize("change,word", BAD_ADAPTERS, ids=str)
def test_adapter_params_refused(nxg, L, change, word):
    p = adapter_params(nxg, **change)
    refused(nxg, L, adapter(nxg, L, p), word)
    refused(nxg, L, adapter_back(nxg, L, p, n=1 << 40), word)
    assert L.nxg_adapter_rows_backward_workspace_bytes(ctypes.byref(p)) == -nxg.NXG_EINVAL


def test_adapter_arrays_refused(nxg, L):
    for change in ({"cu": None}, {"ids": None}, {"a": None}, {"b": None}):
        refused(nxg, L, adapter(nxg, L, adapter_params(nxg, **change)), "null cu, ids, a or b")
        refused(nxg, L, adapter_back(nxg, L, adapter_params(nxg, **change)), "null cu, ids, a or b")
    refused(nxg, L, adapter(nxg, L, adapter_params(nxg, a=P16 + 8)), "a and b must be 16-byte")
    for kw, word in (({"x": None}, "x is null"), ({"x": P16 + 1}, "x is null or not aligned"), ({"base": P16 + 1}, "base is null or not"), ({"y": None}, "y is null"),
                     ({"xs": -1}, "stride -1 of x"), ({"ys": 127}, "stride 127 of y"), ({"s": None}, "s is null"), ({"s": P16 + 2}, "s is null or not"),
                     ({"y": 4 * P16, "ys": 256}, "another stride"), ({"y": 3 * P16}, "another tensor"), ({"s": 3 * P16}, "another tensor"), ({"s": 4 * P16}, "another tensor"),
                     ({"s": 5 * P16}, "another tensor")):
        refused(nxg, L, adapter(nxg, L, **kw), word)
    assert adapter(nxg, L, adapter_params(nxg, T=0)) == nxg.NXG_OK and adapter(nxg, L, adapter_params(nxg, n_seqs=0)) == nxg.NXG_OK
    refused(nxg, L, L.nxg_adapter_rows(None, None, 0, None, 0, None, 0, None, None), "null params")


def test_adapter_backward_refused(nxg, L):
    for kw, word in (({"dy": None}, "dy is null"), ({"x": None}, "x is null"), ({"s": None}, "s is null"), ({"base": P16 + 1}, "base is null or not"), ({"dx": P16 + 1}, "dx is null or not"),
                     ({"dxs": 60}, "stride 60 of dx"), ({"dx": 6 * P16, "dxs": 128}, "another stride"), ({"dx": 3 * P16}, "dx is another"), ({"dx": 4 * P16}, "dx is another"),
                     ({"dx": 5 * P16}, "dx is another"), ({"da": P16 + 1}, "da or db is not aligned"), ({"da": 9 * P16}, "da or db is another"), ({"da": 3 * P16}, "da or db is another"),
                     ({"db": 7 * P16}, "da or db is another"), ({"db": 2 * P16}, "da or db is another"), ({"ws": None}, "workspace"), ({"ws": P16 + 8}, "workspace"), ({"n": 1000}, "workspace")):
        refused(nxg, L, adapter_back(nxg, L, **kw), word)
    assert adapter_back(nxg, L, dx=None, da=None, db=None, ws=None, n=0) == nxg.NXG_OK


def test_adapter_workspace_sizes(nxg, L):
    """Room for s' gradient, the weights turned round, and a part of the sums for each chunk: rising with every size."""
    def size(**kw):
        return L.nxg_adapter_rows_backward_workspace_bytes(ctypes.byref(adapter_params(nxg, **kw)))
    for kw in ({}, {"T": 0}, {"n_seqs": 0}, {"T": 100000}):
        p = adapter_params(nxg, **kw)
        assert size(**kw) >= 4 * p.T * p.rank + 2 * p.n_adapters * p.rank * (p.n_in + p.n_out)
    assert size(T=0, n_adapters=3) < size(T=0, n_adapters=300) and size(rank=16) < size(rank=128) and size(n_in=64) < size(n_in=4096)


def test_host_tensors_refused(nxg):
    """No CPU fallback: tensors that are not on the current device raise."""
    torch = pytest.importorskip("torch")
    x, q, w = torch.zeros(4, 8), torch.zeros(4, 2, 64), torch.zeros(64)
    with pytest.raises(ValueError, match="current device"):
        nxg.dropout_rows(x, 0.1, 1)
    with pytest.raises(ValueError, match="current device"):
        nxg.qk_norm_rope_rows(q, q, w, w, torch.zeros(32, dtype=torch.float64), [0, 4])
    with pytest.raises(ValueError, match="current device"):
        nxg.adapter_rows(x, torch.zeros(1, 4, 8), torch.zeros(1, 8, 4), [0, 4], [0])
    with pytest.raises(ValueError, match="does not take"):
        nxg.adapter_rows(x.double(), torch.zeros(1, 4, 8), torch.zeros(1, 8, 4), [0, 4], [0])


def test_adapter_backward_launches_refused(nxg, L):
    """More strips of 64 columns than a launch of 1,024 threads each takes: refused, not left to the launch."""
    for kw in ({"n_adapters": 131072, "rank": 3, "n_in": 1024, "n_out": 1024}, {"n_adapters": 2097152, "rank": 1, "n_in": 64, "n_out": 64}):
        p = adapter_params(nxg, **kw)
        refused(nxg, L, adapter_back(nxg, L, p, dys=1024, xs=1024, bs=1024, dxs=1024, n=1 << 50), "too large")
