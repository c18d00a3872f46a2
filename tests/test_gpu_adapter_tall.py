"""GPU: adapter_rows' tiles of 64 and 128 rows, which launches of many rows of larger ranks take, against 64 bits: every number of ranks
they are built for, ranks off 16 bytes, several steps of the contracted index and blocks of columns with what is left."""
from __future__ import annotations

import pytest

from test_gpu_adapter_rows import TYPES, Case, dev, torch  # noqa: F401

pytestmark = pytest.mark.gpu

# rows from which on ranks up to 64, and others, take tiles of 64; ranks over 64 tiles of 128
MANY, MOST = 33100, 65700


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("r,T", [(20, MANY), (32, MANY), (40, MANY), (48, MANY), (64, MANY), (65, MANY), (100, MANY), (128, MANY), (72, MOST), (100, MOST), (128, MOST)])
@pytest.mark.parametrize("K,N", [(200, 136), (64, 72)])
def test_tall_tiles(nxg, torch, dev, dtype, wtype, r, T, K, N):  # noqa: F811
    print(f"adapter_rows {dtype} {wtype} r={r}, {T} rows, {K} to {N}", flush=True)
    lens = [T // 2 + 11, 130, 1, 0, T // 4 - 77, T // 8]
    c = Case(torch, dtype, wtype, lens, [1, -1, 2, 0, 0, 1], 3, r, K, N, T=T)
    assert T // len(lens) >= 128
    c.check(nxg, torch)


@pytest.mark.parametrize("dtype,wtype", TYPES)
@pytest.mark.parametrize("r", [48, 128])
def test_tall_tiles_strided_in_place(nxg, torch, dev, dtype, wtype, r):  # noqa: F811
    """Rows inside others, over the base, and rows behind the documents left as they were: the same bits."""
    print(f"adapter_rows {dtype} {wtype} r={r}, {MOST} strided rows in place", flush=True)
    T, K, N = MOST, 72, 88
    c = Case(torch, dtype, wtype, [T - 5000, 400, 4500], [1, -1, 0], 2, r, K, N, T=T)
    y, s = c.forward(nxg)
    dx = c.backward(nxg, s)[0]
    n = int(c.cu[-1])

    def inside(t):
        rows = torch.full((T, t.shape[1] + 24), 7.0, dtype=t.dtype, device="cuda")
        rows[:, 8:8 + t.shape[1]] = t
        return rows, rows[:, 8:8 + t.shape[1]]
    before = c.base[n:].clone(), c.dx_base[n:].clone()
    bufs = {}
    for name in ("x", "dy", "base", "dx_base"):
        bufs[name], t = inside(getattr(c, name))
        setattr(c, name, t)
    s2 = torch.full_like(s, 7.0)
    c.forward(nxg, out=c.base, s=s2)
    c.backward(nxg, s2, dx=c.dx_base)
    assert torch.equal(c.base[:n], y[:n]) and torch.equal(s2[:n], s[:n]) and torch.equal(c.dx_base[:n], dx[:n])
    assert torch.equal(c.base[n:], before[0]) and torch.equal(c.dx_base[n:], before[1]) and (s2[n:] == 7).all()
    for name, rows in bufs.items():
        assert (rows[:, :8] == 7).all() and (rows[:, -16:] == 7).all(), name
