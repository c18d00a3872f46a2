"""GPU: every tile of every document is taken, whatever the order of a launch's workgroups: as many documents as a
wave has lanes and about as many, all of them with rows, in calls of more workgroups than run at once (which are ordered by
their work). Outputs hold NaN before the call, so that a row which is not written shows."""
from __future__ import annotations

import math

import numpy as np
import pytest

import rows_ref

pytestmark = pytest.mark.gpu

LENGTHS = {"mixed": lambda n: [(37 * i) % 150 + 1 for i in range(n)],
           "alike": lambda n: [300] * n,
           "one_short": lambda n: [260] * (n - 1) + [140]}


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.fixture(scope="module")
def dev(torch, nxg):
    nxg.init()
    return torch.device("cuda:0")


@pytest.mark.parametrize("left,right", [(-1, 0), (9, -1), (-1, -1)])
@pytest.mark.parametrize("kind", list(LENGTHS))
@pytest.mark.parametrize("n", [2, 33, 63, 64, 65])
def test_every_document_is_written(nxg, torch, dev, n, kind, left, right):
    print(f"attention_rows {n} documents, {kind}, window={left},{right}", flush=True)
    lens = LENGTHS[kind](n)
    H = G = 8 if n > 2 else 160
    D, T = 16, sum(lens)
    wgs = (T // 128 + n) * G
    assert wgs > 512 or kind == "mixed", "more workgroups than run at once"
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k, v, do = (torch.randn(T, H, D, device="cuda", generator=g).bfloat16() for _ in range(4))
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    out, dq, dk, dv = (torch.full_like(q, math.nan) for _ in range(4))
    lse = torch.full((T, H), math.nan, device="cuda")
    nxg.attention_rows(q, k, v, cu, left=left, right=right, out=out, lse=lse)
    nxg.attention_rows_backward(do, q, k, v, out, lse, cu, left=left, right=right, dq=dq, dk=dk, dv=dv)
    for name, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        lost = [d for d in range(n) if bool(torch.isnan(t[cu[d]:cu[d + 1]]).any())]
        assert not lost, f"{name}: documents {lost} have rows that were not written"
    # the values: of two heads (a head's rows depend on its own alone), against 64 bits
    h = slice(0, 2)
    ref = rows_ref.attention(q[:, h], k[:, h], v[:, h], cu, cu, 1 / math.sqrt(D), left, right, do[:, h])
    for name, t in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        rows_ref.check(name, t[:, h], *ref[name])
