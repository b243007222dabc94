"""The float32 GELU far below zero: its tail's bound without room for an exponent that
is rounded (which at u = -13 would alone be 2^-24 u^2 = 170 roundings)."""
import pytest
import torch

import kernel
from train_cases import DEV, F32, HALF, U, cdf, close, held, pdf

pytestmark = pytest.mark.gpu

# Relative error of the tail Phi(-a) = e t P(t) in units of 2^-24, the worst a's sum:
#   1    the fit, with its coefficients in float32 (5.5e-8)
#   6.8  t = rcp(1 + c a): a rounding and an ulp of the reciprocal (two units), three
#        in all, times d ln(t P) / d ln t, at most 2.28
#   2.9  the Horner steps' roundings, each relative to its partial sum
#   3    e: an ulp of the exponential, and the rounding of the sum that gives it back
#        what the square and the product lost (to 2^-40 of its exponent)
#   2    the products t e and P (t e)
# together 15.6 where they meet.
TAIL = 16 * U


def _arguments():
    x = torch.cat([torch.linspace(-13, 0, 200001, device=DEV), torch.linspace(0, 14, 50001, device=DEV),
                   -torch.logspace(-6, 1.11, 50001, device=DEV)])
    return x.view(1, -1)


def test_forward():
    x = _arguments()
    z = x.double()
    want = z * cdf(z)
    above = (z > 0) * 1.0
    # for z > 0 the tail is taken from 1: one more rounding; results under 2^-120 may be zero
    tol = z.abs() * (TAIL * cdf(-z.abs()) + above * U * cdf(z)) + HALF[F32] * want.abs() * (1 + 1e-5) + 2.0 ** -120
    for t in (x, x.clone().requires_grad_()):
        close(kernel.gelu_packed(t).detach(), want, tol, "gelu")


def test_slope():
    """At held values: Phi(h) + h phi(h), phi with the exponential's 3 units, the
    constant's, and two products'; a rounding of the sum and of its product with dy."""
    x = held(_arguments()).float()
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(kernel.gelu_packed(leaf), leaf, torch.ones_like(x))
    z = held(x)
    assert torch.equal(z.float(), x)
    want = cdf(z) + z * pdf(z)
    above = (z > 0) * 1.0
    tol = TAIL * cdf(-z.abs()) + above * U * cdf(z) + 6 * U * z.abs() * pdf(z) + 2 * U * want.abs() * (1 + 1e-5) + 2.0 ** -120
    close(dx, want, tol, "slope")
