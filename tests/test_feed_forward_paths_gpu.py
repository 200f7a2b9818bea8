"""The feed-forward operators where the other tests do not reach: operands in two layouts, tiles behind the first
of a CTA pair, every tile width, values at the ends of a type's range, calls of several threads.  Against the
definitions in 64 bits; the tolerances are those of test_feed_forward_gpu.py."""

import pytest

torch = pytest.importorskip("torch")

from test_feed_forward_gpu import (F, TYPES, act64, check, dact64, half, normal, own_error, product_slack,  # noqa: E402,F401
                                   weight, SLOPE)

pytestmark = pytest.mark.gpu


def gated_backward64(dh, x, wg, wu, g, u, name):
    """(wanted, slack) of dx, dw_gate, dw_up."""
    dtype, (M, N), K = dh.dtype, dh.shape, x.shape[1]
    g64, u64, dh64 = g.double(), u.double(), dh.double()
    dg, du = dh64 * u64 * dact64(g64, name), dh64 * act64(g64, name)
    h, tiny = half(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    own = own_error(g64, dtype)
    eg = (dh64 * u64).abs() * own + h * dg.abs() * 1.01 + 2.0 ** -22 * dg.abs() + tiny
    eu = dh64.abs() * own + h * du.abs() * 1.01 + 2.0 ** -22 * du.abs() + tiny
    a, b = wg.double().t(), wu.double().t()
    both = product_slack(dg, eg, a, N) + product_slack(du, eu, b, N)
    both = both + (N + 2) * 2.0 ** -23 * (dg.abs() @ a.abs() + du.abs() @ b.abs())
    x64 = x.double()
    return ((dg @ a + du @ b, both), (x64.t() @ dg, product_slack(dg.t(), eg.t(), x64, M).t()),
            (x64.t() @ du, product_slack(du.t(), eu.t(), x64, M).t()))


@pytest.mark.parametrize("element", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layouts", [("kn", "nk"), ("nk", "kn")], ids=str)
def test_gated_weights_in_two_layouts(F, element, layouts):
    dtype = TYPES[element]
    for M, K, N in ((24, 40, 56), (140, 264, 136), (33, 65, 31)):
        x, dh, g, u = normal(M, K, dtype=dtype), *(normal(M, N, dtype=dtype) for _ in range(3))
        wg, wu = (weight(K, N, dtype, layout) for layout in layouts)
        got = F.gated_linear_backward(dh, x, wg, wu, g, u, activation="silu")
        for t, w, (want, slack) in zip(got, (x, wg, wu), gated_backward64(dh, x, wg, wu, g, u, "silu")):
            check(t, want, slack)
            assert t.stride() == w.stride()
