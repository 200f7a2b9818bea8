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
