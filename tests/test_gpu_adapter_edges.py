"""GPU: adapter_rows and adapter_rows_backward at the edges of their sizes: no rows, gradients inside other tensors."""
from __future__ import annotations

import ctypes

import pytest

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
