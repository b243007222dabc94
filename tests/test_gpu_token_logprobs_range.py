"""Token log probabilities of logits far from zero against float64: finite mask
values of any size, rows that hold nothing else, and maxima around the size
from which exponents are formed as differences."""
import math

import pytest
import torch

import kernel
from decode_cases import HALF_STEP

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _reference(x, t, top, scale):
    """(logp, entropy, top indices, top logp, log softmax) in float64, each row
    relative to its maximum (a float64 log-sum-exp near -1e20 has steps of
    16384, and would lose the logarithm)."""
    d = (x.double() - x.double().amax(-1, keepdim=True)) * scale
    lq = d - torch.log(torch.exp(d).sum(-1, keepdim=True))
    ent = -(lq.exp() * lq.clamp(min=-1e30)).sum(-1)
    idx = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    return lq.gather(1, t[:, None])[:, 0], ent, idx, lq.gather(1, idx), lq


def _check(x, t, top=4, scale=1.0):
    """logp, entropy, alternatives and gradient, with the bounds that
    test_gpu_token_logprobs.py derives (2^-17 of max(|value|, log V, 1); the
    gradient's terms there)."""
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda(), top=top, entropy=True, scale=scale)
    logp, ent, idx, tlp, lq = _reference(x, t, top, scale)
    base = max(1.0, math.log(x.size(1)))
    for got, want in ((r.logp, logp), (r.entropy, ent), (r.top_logp, tlp)):
        got = got.detach().double().cpu()
        tol = 2.0 ** -17 * torch.clamp(want.abs(), min=base)
        assert bool(((got - want).abs() <= tol).all()), (got, want)
    assert torch.equal(r.top_index.cpu(), idx)
    g, ge = torch.linspace(-1.5, 1.0, x.size(0)), torch.linspace(0.7, -0.4, x.size(0))
    (dx,) = torch.autograd.grad([r.logp, r.entropy], xg, [g.cuda(), ge.cuda()])
    p = lq.exp()
    want = -g.double()[:, None] * p
    want[torch.arange(len(t)), t] += g.double()
    want = (want - ge.double()[:, None] * p * (lq.clamp(min=-1e30) + ent[:, None])) * scale
    tol = (HALF_STEP[x.dtype] + 3 * 2.0 ** -24) * want.abs() + scale * (2.0 ** -16 * 40.0 * p + 2.0 ** -22 * (p > 0.01)) + 1e-37
    assert bool(((dx.double().cpu() - want).abs() <= tol).all())


MASKS = [-1e4, -1e9, -1e10, -3e10, -1e20, -1e30, -5e37, -3e38]


@pytest.mark.parametrize("value", MASKS)
@pytest.mark.parametrize("R,V", [(3, 50), (3, 5000), (3, 40000), (3, 160000), (600, 4097), (300, 40000)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_mask_values(R, V, dtype, value):
    """A padded vocabulary, a few allowed tokens, and nothing but the mask's
    value (a uniform row)."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(3, V, generator=g) * 2.5).to(dtype)
    x[0, V - V // 9:] = value
    keep = torch.randint(0, V, (6,), generator=g)
    few = torch.full((V,), value).to(dtype)
    few[keep] = x[1, keep]
    x[1] = few
    x[2] = value
    t = torch.tensor([1, int(keep[0]), V - 1])
    x, t = x.repeat(R // 3, 1), t.repeat(R // 3)
    _check(x, t)


@pytest.mark.parametrize("value", [1e10, 3e10, 1e30, 3e38])
def test_large_maximum(value):
    """One token far above the rest, and a uniform row of such values."""
    x = torch.randn(2, 3000, generator=torch.Generator().manual_seed(1))
    x[0, 77] = value
    x[1] = value
    _check(x, torch.tensor([77, 5]))


@pytest.mark.parametrize("middle", [0.0, 65536.0, 11629080.0, 11629080.0 * 2, 1e9])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_maxima_of_any_size(middle, order):
    """Rows of whole steps around `middle` (11629080 log2 e = 2^24): running
    maxima that cross the size, on either side of zero."""
    V = 20000
    step = max(1.0, 2.0 ** (math.frexp(middle)[1] - 24))
    base = torch.arange(V) // (V // 40)
    if order == "down":
        base = base.flip(0)
    elif order == "mixed":
        base = base[torch.randperm(V, generator=torch.Generator().manual_seed(2))]
    x = torch.stack([middle + (base - 20) * step, -middle + (base - 20) * step])
    _check(x, torch.tensor([3, V - 2]), scale=0.75 / step)


def test_large_scale():
    """A scale (inverse temperature) that puts ordinary logits there."""
    x = torch.arange(700).float().remainder(37)[None] * 2.0 ** -20
    _check(x, torch.tensor([36]), scale=float(2 ** 20))
    x = (torch.randn(2, 700, generator=torch.Generator().manual_seed(3)) * 3).to(FP16)
    _check(x, x.float().argmax(-1), scale=3000.0)
