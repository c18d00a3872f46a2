"""GPU: many empty documents between two rows change neither the rows' positions nor, but for a few steps of a search, the time."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.fixture(scope="module")
def dev(torch, nxg):
    nxg.init()
    return torch.device("cuda:0")


def fastest_ms(torch, call):
    """The fastest of five calls, on the GPU's clock."""
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


T = 16384


def calls(nxg, torch, **by):
    """Each operator that finds its rows' places, by offsets or by positions, over the same rows."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, dq, dk = (torch.randn(T, n, 64, device="cuda", generator=g).to(torch.bfloat16) for n in (16, 8, 16, 8))
    w = torch.rand(64, device="cuda", generator=g) + 0.5
    freq = torch.from_numpy(10000.0 ** (-np.arange(32) / 32)).cuda()
    return [lambda: (nxg.rope_rows(q, freq, **by),), lambda: nxg.qk_norm_rope_rows(q, k, w, w, freq, **by),
            lambda: nxg.qk_norm_rope_rows_backward(dq, dk, q, k, w, w, freq, **by)]


@pytest.mark.parametrize("empty", [1, 2, 3, 62, 63, 64, 65, 1000, 20000])
@pytest.mark.parametrize("where", [1, 8193, 16383])
def test_positions_behind_empty_documents(nxg, torch, dev, empty, where):
    print(f"{empty} empty documents in front of row {where}", flush=True)
    cu, plain = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in ([0] + [where] * (empty + 1) + [T], [0, where, T]))
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    pos[where:] -= where
    for call, same, without in zip(calls(nxg, torch, cu_offsets=cu), calls(nxg, torch, positions=pos), calls(nxg, torch, cu_offsets=plain)):
        assert all(torch.equal(a, b) for a, b in zip(call(), same()))
        slow, fast = fastest_ms(torch, call), fastest_ms(torch, without)
        # a search of 2 log2(20,000) = 29 loads at most, of about 1 us each, for a workgroup
        assert slow < 3 * fast + 0.05, (slow, fast)
