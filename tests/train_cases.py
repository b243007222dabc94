"""Inputs, 64-bit definitions and error bounds of the training operators' tests.

EPS[t] / 2 bounds one rounding to t relative to the value; U = 2^-24 that of a
float32 operation.  Bounds on sums count one U per addition on the longest path
of a term."""
import math

import torch

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (BF16, F16, F32)}
# half of the smallest step of a type around zero
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}


def rnd(*shape, seed, std=1.0, dtype=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(shape, device=DEV, dtype=F32).normal_(0.0, std, generator=g).to(dtype)


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise; NaNs where both have them."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    d = (got.double() - want.double()).abs()
    bad = ~((d <= tol) | (got.isnan() & want.isnan()) | (got.double() == want.double()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst excess {float((d - tol)[bad].max()):.3e}"


def in_use():
    """Bytes that the live tensors asked for.  memory_allocated() counts the blocks that
    serve them: a free one that is up to 1 MiB larger is handed out whole, so what it
    shows depends on what ran before."""
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


# ---- LayerNorm --------------------------------------------------------------------

def norm_exact(x, delta, w, b, eps, dy=None, dr=None):
    """(r, y, dx, dw, db) in 64 bits of the rounded r, and their float32 error bounds
    without the final rounding.

    A row's sums are at most 32 terms a thread, then at most 11 additions across
    threads: n = 48 counts them and the divisions.  With M = mean |r|,
    the mean is off by n U M, the variance by (n + 4) U relative beyond that (the
    mean's error enters the centred sum in second order and as C (dm)^2, covered by
    D^2 of the difference), so xh by D = U (n M rstd + n |xh|)."""
    r = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    z, w64 = r.double(), w.double()
    C = z.size(-1)
    m = z.mean(-1, keepdim=True)
    var = (z - m).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (z - m) * rstd
    n = 48
    D = U * n * (z.abs().mean(-1, keepdim=True) * rstd + xh.abs())
    y = xh * w64 + (0 if b is None else b.double())
    out = [r, y, None, None, None]
    tol = [0.0, w64.abs() * D + 2 * U * y.abs(), None, None, None]
    if dy is not None:
        g = dy.double() * w64
        mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = rstd * (g - mg - xh * mgx) + (0 if dr is None else dr.double())
        ga, gx = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
        Dm = (g.abs() * D).mean(-1, keepdim=True)
        tdx = rstd * (U * n * (g.abs() + ga + xh.abs() * gx) + D * mgx.abs() + xh.abs() * Dm) \
            + (rstd * (g - mg - xh * mgx)).abs() * U * n + 2 * U * dx.abs()
        # a channel's sum: at most R / (rows in flight) additions, R bounds it
        R = z.size(0)
        dw, db = (dy.double() * xh).sum(0), dy.double().sum(0)
        tdw = U * (R + n) * (dy.double() * xh).abs().sum(0) + (dy.double().abs() * D).sum(0)
        tdb = U * (R + n) * dy.double().abs().sum(0)
        out[2:] = [dx, dw, db]
        tol[2:] = [tdx, tdw, tdb]
    return out, tol


# ---- 8-bit activations ------------------------------------------------------------------

def held(x):
    """The values that 8 bits stand for, from the definition, in 64 bits."""
    z = x.detach().double()
    C = z.size(-1)
    t = torch.nn.functional.pad(z, (0, -C % 32)).unflatten(-1, (-1, 32))
    m = t.abs().amax(-1, keepdim=True)
    fin = torch.isfinite(t).all(-1, keepdim=True)
    e = torch.frexp(torch.where(fin, m, torch.ones_like(m))).exponent - 1 - 6
    e = torch.where(m > 0, e, torch.full_like(e, -127)).clamp(min=-127).long()
    step = ((e + 1023) << 52).view(torch.float64)
    h = torch.round(t / step).clamp(-127, 127) * step
    return torch.where(fin, h, torch.full_like(h, float("nan"))).flatten(-2)[..., :C]


def cdf(z):
    return torch.special.erfc(z * -math.sqrt(0.5)) / 2


def pdf(z):
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def gelu_tol(z, dtype):
    """Error of z Phi(z) before its rounding.  The tail Phi(-|z|) is off relatively
    by the fit (9.2e-6, 16-bit types; 16 U, float32), by the rounding
    of its exponent z^2 / 2 (z^2 U, twice: the square and the product) and a few
    operations; for z > 0 the tail is subtracted from 1 (one U of the result).
    Results under 2^-120 may be zero."""
    fit = 16 * U if dtype == F32 else 9.2e-6
    return z.abs() * (cdf(-z.abs()) * (fit + (2 * z * z + 8) * U) + 2 * U * cdf(z)) + 2.0 ** -120


def slope_tol(z, dtype):
    """The same of Phi(z) + z phi(z): the tail's error as above, z phi(z)'s that of
    its exponential and a few operations, two more for the sum."""
    fit = 16 * U if dtype == F32 else 9.2e-6
    return cdf(-z.abs()) * (fit + (2 * z * z + 8) * U) + z.abs() * pdf(z) * (2 * z * z + 16) * U + 2 * U * 1.2
