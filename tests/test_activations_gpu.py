"""The activations of the feed-forward operators over their whole range, kernel by kernel, against 64 bits.

A product with a single non-zero term hands each value to the activation unchanged.  Which kernel takes it is
chosen by the operands: x [M, 1] runs on the CTA pairs (16-bit; f32 on its few-row or batch kernel), x [M, 64]
on the few-row kernel where M is small, an x that starts two bytes off an aligned address with K < 33 on the
CUDA cores."""

import math

import pytest

torch = pytest.importorskip("torch")

from tmtest import require_gpu  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def F():
    require_gpu()
    from triton_metal import functional
    yield functional
    functional.release()


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal: what a result may lose to underflow."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def values(dtype, low, high, count=1500):
    return torch.linspace(low, high, count, dtype=torch.float64).to(dtype).unique().cuda()


def forward(F, z, name, kernel, **kw):
    """act(z), each element through a product on `kernel`."""
    M, dtype = z.numel(), z.dtype
    if kernel == "pairs":
        return F.linear(z.view(M, 1), torch.ones(1, 8, device="cuda", dtype=dtype), activation=name, **kw)[:, 0]
    if kernel == "few rows":
        out = []
        for part in z.split(48):
            x = torch.zeros(part.numel(), 64, device="cuda", dtype=dtype)
            x[:, 0] = part
            out.append(F.linear(x, torch.ones(64, 128, device="cuda", dtype=dtype), activation=name, **kw)[:, 0])
        return torch.cat(out)
    x = torch.empty(M * 2 + 1, device="cuda", dtype=dtype)[1:].view(M, 2)
    x.copy_(torch.stack([z, torch.zeros_like(z)], 1))
    w = torch.ones(2, 8, device="cuda", dtype=dtype)
    return F.linear(x, w, activation=name, **kw)[:, 0]


def derivative(F, z, name):
    """act'(z): the gradient of a product with 1, from a gradient of 1."""
    M, one = z.numel(), torch.ones(1, 1, device="cuda", dtype=z.dtype)
    return F.linear_backward(one.expand(M, 1), z.view(M, 1), one, z.view(M, 1), activation=name)[0][:, 0]


def phi(z):
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def upper_tail(z):
    return torch.special.erfc(z / math.sqrt(2)) / 2


def within(got, want, allowed):
    error = (got.double() - want).abs()
    over = ~(error <= allowed)
    if over.any():
        i = int(over.nonzero()[0])
        raise AssertionError(f"{int(over.sum())} of {over.numel()} off, first at {i}: got {float(got[i])}, "
                             f"want {float(want[i])}, error {float(error[i])}, allowed {float(allowed[i])}")


# gelu, f32: z/2 erfc(y) with y = -z sqrt(1/2), whose relative error (the constant's and the product's rounding,
# 2 x 2^-24) is magnified at most 2 y^2 + 1 = z^2 + 1 times for y > 0; CUDA states 4 units in the last place
# (4 x 2^-23) for erfcf; one rounding.
def gelu_relative(z):
    return (z * z + 6) * 2.0 ** -23


@pytest.mark.parametrize("kernel", ["pairs", "few rows", "cuda cores"])
def test_gelu_keeps_its_relative_accuracy_for_negative_f32(F, kernel):
    z = values(torch.float32, -12, 0)
    z64 = z.double()
    want = z64 * upper_tail(-z64)
    within(forward(F, z, "gelu", kernel), want, gelu_relative(z64) * want.abs() + tiny(torch.float32))


def test_gelu_derivative_keeps_its_accuracy_for_negative_f32(F):
    """Phi + z phi: each term to the relative accuracy above (expf: 2 units, its argument's rounding magnified
    z^2 / 2 times, three products), one rounding of the sum."""
    z = values(torch.float32, -12, 0)
    z64 = z.double()
    left, right = upper_tail(-z64), z64 * phi(z64)
    within(derivative(F, z, "gelu"), left + right, (z64 * z64 + 8) * 2.0 ** -23 * (left + right.abs()) + tiny(torch.float32))


# gelu, 16 bits: the tail is within 2.2e-5 of itself; its exponential's argument, up to z^2 / 2, is rounded a few
# times (z^2 2^-23), the approximate exponential and quotient add a few units of 2^-23 each; then one rounding.
def fast_tail_relative(z):
    return 2.2e-5 + (z * z + 16) * 2.0 ** -23


@pytest.mark.parametrize("kernel", ["pairs", "few rows", "cuda cores"])
@pytest.mark.parametrize("element", ["f16", "bf16"])
def test_gelu_of_16_bits_is_within_its_rounding_in_the_tail(F, element, kernel):
    dtype = TYPES[element]
    z = values(dtype, -12, 0, 6000)
    z64 = z.double()
    want = z64 * upper_tail(-z64)
    slack = fast_tail_relative(z64) * want.abs()
    within(forward(F, z, "gelu", kernel), want, slack + half(dtype) * (want.abs() + slack) + tiny(dtype))


@pytest.mark.parametrize("element", ["f16", "bf16"])
def test_gelu_derivative_of_16_bits_is_within_its_rounding_in_the_tail(F, element):
    dtype = TYPES[element]
    z = values(dtype, -12, 0, 6000)
    z64 = z.double()
    left, right = upper_tail(-z64), z64 * phi(z64)
    slack = fast_tail_relative(z64) * (left + right.abs())
    want = left + right
    within(derivative(F, z, "gelu"), want, slack + half(dtype) * (want.abs() + slack) + tiny(dtype))


# ---- the ends of the range --------------------------------------------------------------------------------

def act64(z, name):
    """Limits at the infinities for all but silu and gelu_tanh of minus infinity, which are NaN (minus infinity times
    0), as their products of the argument with a sigmoid give."""
    if name == "gelu":
        return torch.where(z == -math.inf, torch.zeros_like(z), torch.where(z < 0, z * upper_tail(-z), z * (1 - upper_tail(z))))
    return {"none": lambda: z, "relu": lambda: torch.where(z < 0, torch.zeros_like(z), z),
            "silu": lambda: z * torch.sigmoid(z), "sigmoid": lambda: torch.sigmoid(z),
            "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[name]()


def dact64(z, name):
    """By formula, with the limits where a factor overflows."""
    s = torch.sigmoid(z)
    inner, slope = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3), math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    t = torch.sigmoid(2 * inner)
    far = z.abs() > 50
    limit = torch.where(z > 0, 1.0, 0.0).double()
    value = {"none": torch.ones_like(z), "relu": limit, "gelu": upper_tail(-z) + z * phi(z), "sigmoid": s * (1 - s),
             "silu": s * (1 + z * (1 - s)), "gelu_tanh": t + z * t * (1 - t) * 2 * slope}[name]
    if name not in ("none", "relu"):
        value = torch.where(far, torch.zeros_like(z) if name == "sigmoid" else limit, value)
    return torch.where(z.isnan() & (name != "none"), z, value)


def ends(dtype):
    f = torch.finfo(dtype)
    sizes = [0.0, f.smallest_normal * f.eps, f.smallest_normal, 1e-4, 0.1, 1.0, 3.0, 10.0, 20.0, 60.0, 85.0, 90.0, 101.0, 300.0,
             6.0e4, f.max ** 0.5, f.max / 2, f.max, math.inf]
    return torch.tensor(sizes + [-v for v in sizes] + [math.nan], dtype=torch.float64).to(dtype).cuda()


def same_ends(got, want, z, slack):
    """Equal where not finite; else within the slack, one rounding, and 1e-36: exp(-z) overflows from z = -88.7 on, and
    what is left of silu there is lost."""
    dtype = got.dtype
    rounded = want.to(dtype).double()
    special = ~torch.isfinite(rounded)
    assert torch.equal(got.double()[special].nan_to_num(nan=7.0), rounded[special].nan_to_num(nan=7.0)), (z[special], got[special])
    within(got[~special], want[~special], (slack + half(dtype) * (want.abs() + slack) + tiny(dtype) + 1e-36)[~special])


@pytest.mark.parametrize("kernel", ["pairs", "few rows", "cuda cores"])
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_the_ends_of_the_range(F, name, element, kernel):
    z = ends(TYPES[element])
    z64 = z.double()
    out = forward(F, z, name, kernel)
    # a few units of fp32 in the value; the sigmoids' arguments, up to 90 where they matter, are rounded too
    want = act64(z64, name)
    slack = (want.abs() if name != "none" else 0 * z64).nan_to_num(nan=0.0, posinf=0.0, neginf=0.0) * (
        2.0 ** -15 if element != "f32" else 2.0 ** -18)
    same_ends(out, want, z, slack)


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_derivatives_at_the_ends_of_the_range(F, name, element):
    z = ends(TYPES[element])
    want = dact64(z.double(), name)
    # (1 + |z| <= 90 terms of size 1 at most, each within a few units of fp32)
    slack = torch.full_like(want, 2.0 ** -17 if element != "f32" else 2.0 ** -20)
    same_ends(derivative(F, z, name), want, z, slack)


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_gated_product_and_gradient_at_the_ends_of_the_range(F, name, element):
    """One row of gates beside ups of 1: the value, dgate = act'(gate) and dup = act(gate)."""
    dtype = TYPES[element]
    z = ends(dtype)
    n = z.numel()
    one, x = torch.ones(n, 1, device="cuda", dtype=dtype), z.view(n, 1)
    unit = torch.ones(1, 1, device="cuda", dtype=dtype)
    want = act64(z.double(), name)
    slack = want.abs().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0) * (2.0 ** -15 if element != "f32" else 2.0 ** -18)
    # x (w_gate, w_up) = (gate, up) needs an up of its own: the gate in column 0 of two, 1 in the other
    two = torch.cat([x, one], 1)
    wg = torch.tensor([[1.0], [0.0]], device="cuda", dtype=dtype)
    finite = torch.isfinite(z)                                     # (infinity times the 0 of w_up is NaN)
    h = F.gated_linear(two[finite], wg, wg.flip(0), activation=name)
    same_ends(h[:, 0], want[finite], z[finite], slack[finite])
    # dw_up and dx through a unit weight: dx = dgate + dup, with dup removed by a w_up of 0
    zero = torch.zeros_like(unit)
    dgate = F.gated_linear_backward(one, one, unit, zero, x, one, activation=name)[0][:, 0]
    up = F.gated_linear_backward(one, one, zero, unit, x, one, activation=name)[0][:, 0]
    d = dact64(z.double(), name)
    # (a NaN or infinity times that 0 is NaN)
    keep = torch.isfinite(want.to(dtype))
    same_ends(dgate[keep], d[keep], z[keep], torch.full_like(d, 2.0 ** -17 if element != "f32" else 2.0 ** -20)[keep])
    keep = torch.isfinite(d)
    same_ends(up[keep], want[keep], z[keep], slack[keep])
