"""CPU: the 64-bit forms of adapter_ref.py against differentiation, differences and the generator's published vectors."""
from __future__ import annotations

import numpy as np
import pytest

import adapter_ref

torch = pytest.importorskip("torch")


def test_philox_known_answers():
    """The vectors published with the generator: counter, key, result."""
    ones = 0xFFFFFFFF
    for c, k, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                       ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                       ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                        (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in adapter_ref.philox(np.array(c, np.uint64), k)) == want


def test_kept_is_one_draw_a_value():
    a = adapter_ref.kept(40, 30, 0.25, 5, 9)
    assert np.array_equal(a[:17, :11], adapter_ref.kept(17, 11, 0.25, 5, 9))        # by (row, column) alone
    assert not np.array_equal(a, adapter_ref.kept(40, 30, 0.25, 6, 9)) and not np.array_equal(a, adapter_ref.kept(40, 30, 0.25, 5, 10))
    assert not np.array_equal(a, adapter_ref.kept(40, 30, 0.25, 5 + 2 ** 32, 9)) and not np.array_equal(a, adapter_ref.kept(40, 30, 0.25, 5, 9 + 2 ** 32))
    big = adapter_ref.kept(2000, 500, 0.25, 1, 2)
    assert abs(big.mean() - 0.75) < 6 * (0.25 * 0.75 / big.size) ** 0.5
    assert adapter_ref.kept(3, 9, 0.0, 1, 2).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_qk_norm_rope_gradient(layout):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 12, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(12, generator=g, dtype=torch.float64).requires_grad_()
    dy = torch.randn(5, 3, 12, generator=g, dtype=torch.float64)
    f, pos = torch.tensor([1.0, 0.3, 0.01, 0.002], dtype=torch.float64), torch.tensor([0, 4, 9, 1, 2])
    y = adapter_ref.qk_norm_rope(x, w, f, pos, layout, 1.5, 1e-3)[0]
    want = torch.autograd.grad(y, (x, w), dy)
    got = adapter_ref.qk_norm_rope_back(dy, x.detach(), w.detach(), f, pos, layout, 1.5, 1e-3)
    for (v, bound), ref in zip(got, want):
        assert float((v - ref).abs().max()) < 1e-12 and float(bound.min()) > 0


def test_adapter_gradient():
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    cu, ids = [0, 3, 3, 7, 9], [1, 0, 1, -1]
    x, a, b = rnd(10, 6).requires_grad_(), rnd(2, 3, 6).requires_grad_(), rnd(2, 5, 3).requires_grad_()
    dy, base = rnd(10, 5), rnd(10, 6)
    y = torch.stack([0.5 * b[1] @ (a[1] @ x[t]) if t < 7 else 0 * x[t, :5] for t in range(9)])
    (v, _), (s, _) = adapter_ref.adapter(x.detach().float(), a.detach().float(), b.detach().float(), cu, ids, 0.5, None)
    assert float((v[:9] - y.detach()).abs().max()) < 1e-5 and bool(torch.isnan(v[9]).all()) and bool((s[7:9] == 0).all())
    want = torch.autograd.grad(y, (x, a, b), dy[:9])
    s = x.detach() @ a.detach()[1].t()
    with torch.no_grad():
        got = adapter_ref.adapter_back(dy.float(), x.float(), a.float(), b.float(), s.float(), cu, ids, 0.5, base.float())
    assert float((got[0][0][:9] - base[:9] - want[0][:9]).abs().max()) < 1e-5
    for (v, bound), ref in zip(got[1:], want[1:]):
        assert float((v - ref).abs().max()) < 1e-5 and bool((v[0] == 0).all())
