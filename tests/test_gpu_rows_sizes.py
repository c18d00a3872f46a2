"""GPU: sizes and windows past 32 bits, which the row operators' C functions count in, are what they say or refused; never
taken modulo 2^32."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

PAST = (1 << 32) + 5         # 5 in 32 bits


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "no GPU"
    return t


@pytest.mark.parametrize("left,right", [(1 << 32, 0), ((1 << 32) + 3, 1 << 32), (1 << 31, (1 << 33) + 2), (1 << 63, 1 << 40)])
def test_windows_past_32_bits(nxg, torch, left, right):
    print(f"attention_rows window={left},{right}", flush=True)
    nxg.init()
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(90, n, 64, device="cuda", generator=g).bfloat16() for n in (4, 2, 2, 4))
    cu = [0, 50, 90]
    want = dict(left=-1, right=-1 if right else 0)
    got = dict(left=left, right=right)
    a, b = (nxg.attention_rows(q, k, v, cu, **w) for w in (want, got))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a, b = (nxg.attention_rows_backward(do, q, k, v, a[0], a[1], cu, **w) for w in (want, got))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for bad in (-(1 << 32) - 1, -(1 << 32), -2):
        with pytest.raises(ValueError, match="left"):
            nxg.attention_rows(q, k, v, cu, left=bad)
        with pytest.raises(ValueError, match="right"):
            nxg.attention_rows(q, k, v, cu, right=bad)


def test_rows_past_32_bits(nxg, torch):
    """One row repeated more than 2^32 times: refused before anything of that size is made."""
    print("row operators of 2^32 + 5 rows", flush=True)
    nxg.init()
    x = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda").expand(PAST, 1)
    q = torch.ones(1, 1, 8, dtype=torch.bfloat16, device="cuda").expand(PAST, 1, 8)
    short = torch.ones(5, 1, 8, dtype=torch.bfloat16, device="cuda")
    stat = torch.ones(1, device="cuda").expand(PAST)
    freq = torch.ones(4, dtype=torch.float64, device="cuda")
    used = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for call in (lambda: nxg.layer_norm_rows(x), lambda: nxg.layer_norm_rows_backward(x, x, stat, stat),
                 lambda: nxg.rope_rows(q, freq, [0, 5]), lambda: nxg.attention_rows(q, short, short, [0, 5]),
                 lambda: nxg.attention_rows(short, q, q, [0, 5]),
                 lambda: nxg.attention_rows_backward(q, q, short, short, q, stat[:, None], [0, 5]),
                 lambda: nxg.attention_rows_backward_workspace_bytes(q, q, q, [0, 5]),
                 lambda: nxg.layer_norm_rows_workspace_bytes(PAST, 64), lambda: nxg.layer_norm_rows_workspace_bytes(64, PAST)):
        with pytest.raises(ValueError):
            call()
    assert torch.cuda.max_memory_allocated() < used + (1 << 20)


def test_frequencies_past_32_bits(nxg):
    for args in (((1 << 32) + 64, 1e4), (64, 1e4, "by_parts", 2.0, (1 << 32) + 1)):
        with pytest.raises(ValueError):
            nxg.rope_frequencies(*args)
