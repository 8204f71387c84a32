"""The gradient norm over the range of its types, against squares in float64.

Tolerance of the norm: a thread adds at most 64 squares per chunk in float32, each product
and sum off by 2^-24, so its sum by 64 2^-24 and the norm by half of that, 2e-6; the result's
own rounding is 2^-24, or half the smallest float32 (2^-150) where the norm itself is
subnormal."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def norm64(grads):
    # (float64 holds the squares of every float32 down to 2^-149: 2^-298)
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-14, 1e-17, 1e-19, 1e-21, 1e-24, 1e-36, 1e-39])
@pytest.mark.parametrize("n,start", [(1, 0), (40003, 0), (16384, 0), (5000, 1)])
def test_small_elements(dtype, size, n, start):
    """Elements whose squares are subnormal in float32, or zero."""
    from evograd_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.randn(n + start, device="cuda", generator=g, dtype=torch.float64) * size).to(dtype)[start:]
    want = norm64([x])
    assert want > 0
    got = float(ops.grad_norm([x]))
    assert abs(got - want) <= 2e-6 * want + 2.0 ** -150, (got, want)


def test_small_elements_beside_others():
    """Each thread's sum has the bits its own elements need: all zeros, small ones, and one
    tensor of ordinary size that makes the small ones invisible."""
    from evograd_b200 import ops

    z = torch.zeros(100000, device="cuda")
    small = torch.full((70001,), 3e-23, device="cuda")
    one = torch.zeros(50000, device="cuda")
    one[777] = 2e-22
    want = norm64([small, one])
    assert abs(float(ops.grad_norm([z, small, one])) - want) <= 2e-6 * want
    assert float(ops.grad_norm([z])) == 0.0
    big = torch.ones(16, device="cuda")
    assert abs(float(ops.grad_norm([z, small, one, big])) - 4.0) <= 1e-5


def test_scaling_by_a_small_norm():
    """max_norm as small as the gradients: the factor's denominator is the 1e-6 of the formula."""
    from evograd_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(30000, device="cuda", generator=g) * 1e-21
    keep, want = x.double(), norm64([x])
    norm = ops.clip_grad_norm([x], want / 4)
    assert abs(float(norm) - want) <= 2e-6 * want
    coef = min(1.0, want / 4 / (want + 1e-6))
    assert bool(((x.double() - keep * coef).abs() <= 2.0 ** -22 * keep.abs() * coef + 2.0 ** -149).all())


def test_norm_beyond_float32():
    """The returned float32 is infinite where the norm is beyond float32; the scaling goes by
    the float64 norm."""
    from evograd_b200 import ops

    x = torch.full((100,), 3e38, device="cuda")
    norm = ops.clip_grad_norm([x], 1.0)
    assert math.isinf(float(norm))
    # 0.1, off by the roundings of a float32 factor (subnormal: 2^-150 of 3e-40) and the product
    factor = 1.0 / (10 * float(torch.tensor(3e38)))
    slack = 2.0 ** -150 / factor + 2.0 ** -22
    assert bool(((x.double() - 0.1).abs() <= 0.1 * slack).all())
