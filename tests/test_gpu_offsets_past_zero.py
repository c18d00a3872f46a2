"""GPU: device offsets that do not start at 0 give unspecified rows but no access out of bounds."""
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


@pytest.mark.parametrize("first", [4000, 6000])
def test_attention_rows_many_documents(nxg, torch, dev, first):
    """More documents than a wave has lanes, the first of them behind a slot's: looked for by their offsets."""
    print(f"attention_rows, 100 documents from row {first}", flush=True)
    T = 6000
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, dout = (torch.randn(T, n, 64, device="cuda", generator=g).to(torch.bfloat16) for n in (4, 2, 2, 4))
    cu = torch.tensor(np.linspace(first, T, 101).astype(np.int32), device="cuda")
    for right in (-1, 0):
        out = torch.full((T + 2, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        _, lse = nxg.attention_rows(q, k, v, cu, right=right, out=out[1:T + 1])
        grads = nxg.attention_rows_backward(dout, q, k, v, out[1:T + 1], lse, cu, right=right)
        torch.cuda.synchronize()
        assert (out[0] == 7).all() and (out[T + 1] == 7).all() and grads[0].shape == q.shape
    # the same offsets from 0, with the rows in front as a document of their own: its neighbours' results
    if first < T:
        whole = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), cu])
        want = nxg.attention_rows(q, k, v, whole, right=0)[0]
        assert torch.isfinite(want).all()


@pytest.mark.parametrize("docs", [1, 40, 70])
def test_lily_state_many_rows(nxg, torch, dev, docs):
    """The kernel for many rows, whose first rows lie in front of every document."""
    print(f"lily state, {docs} documents from row 20,000", flush=True)
    T, C = 22001, 1024
    g = torch.Generator(device="cuda").manual_seed(1)
    a, x, b = (torch.randn(T, C, device="cuda", generator=g) for _ in range(3))
    cu = torch.tensor(np.linspace(20000, T, docs + 1).astype(np.int32), device="cuda")
    qa = nxg.lily_state_quantize_rows(a, x, b, torch.randn(2, C, device="cuda", generator=g), cu)
    torch.cuda.synchronize()
    assert qa.T == T


@pytest.mark.parametrize("first,docs", [(4000, 100), (4000, 64), (1, 70), (5990, 3)])
@pytest.mark.parametrize("right", [-1, 0])
def test_attention_rows_of_documents_behind_other_rows(nxg, torch, dev, first, docs, right):
    """The documents' rows are those of a call in which the rows in front are a document of their own, forward and back, and the rows
    in front are left as they were."""
    print(f"attention_rows, {docs} documents from row {first}, against a document in front", flush=True)
    T = 6000
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, dout = (torch.randn(T, n, 64, device="cuda", generator=g).to(torch.bfloat16) for n in (4, 2, 2, 4))
    cu = torch.tensor(np.linspace(first, T, docs + 1).astype(np.int32), device="cuda")
    whole = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), cu])
    want, lse_want = nxg.attention_rows(q, k, v, whole, right=right)
    grads_want = nxg.attention_rows_backward(dout, q, k, v, want, lse_want, whole, right=right)
    out, lse = torch.full_like(q, 7.0), torch.full((T, 4), 7.0, device="cuda")
    nxg.attention_rows(q, k, v, cu, right=right, out=out, lse=lse)
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    nxg.attention_rows_backward(dout, q, k, v, want, lse_want, cu, right=right, dq=grads[0], dk=grads[1], dv=grads[2])
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + tuple(grads), (want, lse_want) + tuple(grads_want)):
        assert (a[:first] == 7).all(), name
        # the two launches may share a long sum out differently: fp32 sums of up to 6,000 terms, rounded to bf16 once
        d = (a[first:].float() - b[first:].float()).abs()
        assert bool((d <= 2.0 ** -7 * b[first:].float().abs() + 6000 * 2.0 ** -24 * b[first:].float().abs().max()).all()), name
