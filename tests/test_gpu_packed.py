"""8-bit activations: what they stand for is defined to the bit, gelu_packed and
mlp_packed follow from it; bounds from train_cases."""
import math

import pytest
import torch
import torch.nn.functional as F

import kernel
from train_cases import BF16, DEV, F16, F32, HALF, LEAST, U, cdf, close, gelu_tol, held, in_use, pdf, rnd, slope_tol

pytestmark = pytest.mark.gpu

TYPES = [BF16, F16, F32]


def _same(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def _spread(R, C, dtype, seed):
    """Values of many sizes: every row and block its own."""
    s = torch.exp2(rnd(R, -(-C // 32), seed=seed + 1, std=2.0)).repeat_interleave(32, 1)[:, :C]
    return (rnd(R, C, seed=seed) * s).to(dtype)


def _check_gelu(x, dy):
    leaf = x.detach().requires_grad_()
    y = kernel.gelu_packed(leaf)
    assert y.shape == x.shape and y.dtype == x.dtype
    z = x.detach().double()
    want = z * cdf(z)
    close(y.detach(), want, gelu_tol(z, x.dtype) + HALF[x.dtype] * want.abs() * (1 + 1e-4) + LEAST[x.dtype], "y")
    (dx,) = torch.autograd.grad(y, leaf, dy)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    h = held(x)
    want = dy.double() * (cdf(h) + h * pdf(h))
    close(dx, want, dy.double().abs() * slope_tol(h, x.dtype) + HALF[x.dtype] * want.abs() * (1 + 1e-4) + LEAST[x.dtype], "dx")
    return y.detach(), dx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,C", [(1, 1), (1, 32), (3, 7), (5, 31), (4, 33), (7, 64), (9, 100), (130, 2048), (33, 4801), (1000, 40)])
def test_values(dtype, R, C):
    x = _spread(R, C, dtype, R + C)
    p = kernel.pack_activation(x)
    assert p.q.shape == x.shape and p.q.dtype == torch.int8 and p.dtype == dtype
    assert p.exp.shape == (R, (C + 31) // 32) and p.exp.dtype == torch.uint8
    want = held(x)
    _same(kernel.unpack_activation(p), want.to(dtype))
    for t in TYPES:
        _same(kernel.unpack_activation(p, dtype=t), want.float().to(t))
    # off by a 128th of the block's largest magnitude at most, in whole steps of it
    m = F.pad(x.double(), (0, -C % 32)).unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, 1)[:, :C]
    assert ((want - x.double()).abs() <= m / 128 + 2.0 ** -128).all()
    # a held activation stands for itself
    _same(kernel.unpack_activation(kernel.pack_activation(want.to(dtype))), want.to(dtype))
    _check_gelu(x, rnd(R, C, seed=9, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_values_at_the_edges(dtype):
    """Zeros, the type's smallest and largest numbers, halves of a step, infinities
    and NaN: a block that is not finite stands for NaN, its neighbours for themselves."""
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    tiny = {BF16: 2.0 ** -133, F16: 2.0 ** -24, F32: 2.0 ** -149}[dtype]
    x = torch.zeros(12, 96, device=DEV, dtype=dtype)
    x[1, 3] = -0.0
    x[2, :40] = tiny
    x[3, ::3] = low
    x[3, 1] = -tiny
    x[4, 5], x[4, 6], x[4, 7] = top, -top, top / 2
    x[5, :32] = torch.arange(32, device=DEV) * 0.5 + 64.5      # halves of a step of 1
    x[5, 0] = 127.5
    x[6, 40] = float("inf")
    x[7, 41] = float("-inf")
    x[8, 0] = float("nan")
    x[9] = 1
    x[10] = torch.linspace(-1, 1, 96)
    want = held(x)
    got = kernel.unpack_activation(kernel.pack_activation(x))
    _same(got, want.to(dtype))
    assert got[6, 32:64].isnan().all() and got[7, 32:64].isnan().all() and got[8, :32].isnan().all()
    assert got[6, :32].isfinite().all() and got[6, 64:].isfinite().all() and got[9:].isfinite().all()
    _check_gelu(x[[0, 1, 2, 3, 5, 9, 10, 11]], rnd(8, 96, seed=1, dtype=dtype))
    leaf = x.requires_grad_()
    y = kernel.gelu_packed(leaf)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(dx.isnan(), want.isnan())
    # the forward pass has the exact values: +inf stays, -inf and NaN give NaN as torch's
    assert y[6, 40] == float("inf") and y[7, 41].isnan() and y[8, 0].isnan() and int(y.isnan().sum()) == 2
    assert dx[4, 5] == 1 and dx[4, 6] == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_all_sizes_of_argument(dtype):
    """The whole curve, its far tails among them."""
    x = torch.cat([torch.linspace(-15, 15, 40000, device=DEV), torch.logspace(-30, 4, 8000, device=DEV),
                   -torch.logspace(-30, 4, 8000, device=DEV)]).to(dtype)
    y, _ = _check_gelu(x[:, None].contiguous(), torch.ones(len(x), 1, device=DEV, dtype=dtype))
    assert y[x[:, None] > 16].eq(x[x > 16][:, None].flatten()).all()


def test_shapes_and_layouts():
    x = _spread(24, 70, BF16, 3)
    dy = rnd(24, 70, seed=4, dtype=BF16)
    want, p = _check_gelu(x, dy), kernel.pack_activation(x)

    def wide(t):
        big = torch.zeros(24, 75, device=DEV, dtype=BF16)
        big[:, 3:73] = t
        return big[:, 3:73]

    for f in (wide, lambda t: t.t().contiguous().t(), lambda t: t.view(2, 3, 4, 70), lambda t: t.view(4, 6, 70)):
        got, q = _check_gelu(f(x), f(dy)), kernel.pack_activation(f(x))
        for a, b in zip((*got, q.q), (*want, p.q)):
            assert torch.equal(a.reshape(b.shape), b)
        assert torch.equal(q.exp.reshape(p.exp.shape), p.exp)
        assert torch.equal(kernel.unpack_activation(q).reshape(24, 70), kernel.unpack_activation(p))
    for a, b in zip(_check_gelu(x[0], dy[0]), want):
        assert torch.equal(a, b[0])
    _check_gelu(x, torch.ones((), device=DEV, dtype=BF16).expand(24, 70))


def test_nothing():
    for shape in ((0, 40), (3, 0, 40), (0, 1)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = kernel.gelu_packed(x)
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert y.shape == g.shape == x.shape
        assert kernel.unpack_activation(kernel.pack_activation(x.detach())).shape == x.shape


def test_rows_past_32_bits():
    R, C = (1 << 19) + 1, 8200
    x = torch.zeros(R, C, device=DEV, dtype=BF16)
    x[-1] = rnd(C, seed=1)
    p = kernel.pack_activation(x)
    assert torch.equal(p.q[-1], kernel.pack_activation(x[-1].clone()).q) and not p.q[1].any()
    y = kernel.unpack_activation(p)
    assert torch.equal(y[-1].double(), held(x[-1:])[0]) and not y[-2].any()
    del y, p
    y = kernel.gelu_packed(x)
    assert torch.equal(y[-1], kernel.gelu_packed(x[-1].clone()))


def test_against_differences():
    """At held values the gradient is that of the GELU: central differences of its
    float32 results (h^2 / 6 of the third derivative, at most 2, and 4 U of values
    up to 4 over 2 h)."""
    x = held(rnd(8, 64, seed=5)).float()
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(kernel.gelu_packed(leaf), leaf, torch.ones_like(x))
    h = 2.0 ** -6
    d = (kernel.gelu_packed(x + h).double() - kernel.gelu_packed(x - h).double()) / (2 * h)
    close(g, d, h * h * 2 / 6 + 4 * U * 4 / h)


def test_no_second_derivative():
    x = rnd(4, 32, seed=1).requires_grad_()
    (g,) = torch.autograd.grad(kernel.gelu_packed(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice differentiating"):
        g.sum().backward()


def test_what_is_kept():
    """The graph of a GELU holds its input's 8 bits and nothing else of it."""
    x = rnd(1 << 12, 1 << 10, seed=1, dtype=BF16)
    leaf = x.requires_grad_()
    torch.cuda.synchronize()
    before = in_use()
    y = kernel.gelu_packed(leaf)
    assert in_use() - before <= y.numel() * (2 + 1 + 1 / 32) + 4096


# ---- the whole MLP ------------------------------------------------------------------

def _mlp_case(dtype, lead, C, Fd, Co, bias, seed=0):
    x = rnd(*lead, C, seed=seed, dtype=dtype)
    ws = [rnd(Fd, C, seed=seed + 1, std=C ** -0.5, dtype=dtype), rnd(Co, Fd, seed=seed + 2, std=Fd ** -0.5, dtype=dtype)]
    bs = [rnd(Fd, seed=seed + 3, std=0.3, dtype=dtype), rnd(Co, seed=seed + 4, std=0.3, dtype=dtype)] if bias else [None, None]
    return x, ws, bs, rnd(*lead, Co, seed=seed + 5, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,C,Fd,Co,bias", [((1,), 8, 32, 8, True), ((2, 33), 64, 256, 64, True), ((130,), 96, 200, 40, False)])
def test_mlp(dtype, lead, C, Fd, Co, bias):
    """Each gradient against the formula of the held activations in 64 bits.  Products
    of K terms: K U of the sum of magnitudes in float32 (library GEMMs of 16-bit types
    accumulate in float32 too), and every stored intermediate one rounding of its type,
    which the next product adds up in magnitude."""
    x, (w1, w2), (b1, b2), gy = _mlp_case(dtype, lead, C, Fd, Co, bias)
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, w1, w2, b1, b2)]
    y = kernel.mlp_packed(*leaves)
    u = F.linear(x, w1, b1)                                  # the very tensor that the operator packs
    E = HALF[dtype] * 1.01
    D = lambda t: t.double().reshape(-1, t.size(-1))          # noqa: E731
    a = D(u) * cdf(D(u))
    da = gelu_tol(D(u), dtype) + E * a.abs() + LEAST[dtype]
    out = a @ D(w2).t() + (0 if b2 is None else b2.double())
    mag = a.abs() @ D(w2).abs().t() + (0 if b2 is None else b2.double().abs())
    close(D(y.detach()), out, da @ D(w2).abs().t() + (Fd + 4) * U * mag + E * out.abs() + LEAST[dtype], "y")
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], gy)
    h, xh, g = held(u).reshape(-1, Fd), held(x).reshape(-1, C), D(gy)
    n = g.size(0)
    ga = g @ D(w2)
    tga = (Co + 4) * U * (g.abs() @ D(w2).abs()) + E * ga.abs() + LEAST[dtype]
    s = cdf(h) + h * pdf(h)
    du = ga * s
    tdu = tga * s.abs() + (ga.abs() + tga) * slope_tol(h, dtype) + E * du.abs() * 1.1 + LEAST[dtype]
    act = h * cdf(h)
    tact = gelu_tol(h, dtype) + E * act.abs() + LEAST[dtype]

    def product(a, ta, b, tb, K):
        ref = a @ b
        return ref, ta @ (b.abs() + tb) + a.abs() @ tb + (K + 4) * U * ((a.abs() + ta) @ (b.abs() + tb)) + E * ref.abs() * 1.1 + LEAST[dtype]

    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    one = torch.ones(1, n, dtype=torch.float64, device=DEV)
    w1d = D(w1)
    refs = [product(du, tdu, w1d, zero.expand_as(w1d), Fd), product(du.t(), tdu.t(), xh, zero.expand_as(xh), n),
            product(g.t(), zero.expand_as(g.t()), act, tact, n)]
    if bias:
        refs += [product(one, zero.expand_as(one), du, tdu, n), product(one, zero.expand_as(one), g, zero.expand_as(g), n)]
    for name, t, (ref, tol) in zip(("dx", "dw_fc", "dw_proj", "db_fc", "db_proj"), got, refs):
        close(t.reshape(ref.shape), ref, tol, name)


def test_mlp_parts():
    """Any inputs that need a gradient; without any, and under no_grad, the same result."""
    x, ws, bs, gy = _mlp_case(F32, (20,), 32, 64, 32, True)
    args = [x, *ws, *bs]
    leaves = [t.detach().requires_grad_() for t in args]
    y = kernel.mlp_packed(*leaves)
    full = torch.autograd.grad(y, leaves, gy)
    for mask in range(1, 32):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
        got = torch.autograd.grad(kernel.mlp_packed(*some), [t for t in some if t.requires_grad], gy)
        for g, i in zip(got, [i for i in range(5) if mask >> i & 1]):
            assert torch.equal(g, full[i]), (mask, i)
    with torch.no_grad():
        assert torch.equal(kernel.mlp_packed(*args), y.detach())
    assert torch.equal(kernel.mlp_packed(*args), y.detach())


def test_mlp_shapes():
    """One row without a leading dimension, no rows at all, weights of other strides."""
    x, ws, bs, gy = _mlp_case(F32, (20,), 32, 64, 32, True)
    leaves = [t.detach().requires_grad_() for t in (x[0], *ws, *bs)]
    y = kernel.mlp_packed(*leaves)
    rows = [t.detach().requires_grad_() for t in (x[:1], *ws, *bs)]
    want = kernel.mlp_packed(*rows)
    assert y.shape == (32,)
    tol = 64 * U * 32                                         # two library products of 64 terms of magnitude up to 4
    close(y.detach(), want.detach()[0], tol)
    for a, b in zip(torch.autograd.grad(y, leaves, gy[0]), torch.autograd.grad(want, rows, gy[:1])):
        close(a.reshape(b.shape), b, tol * 4)
    for lead in ((0,), (3, 0)):
        none = [t.detach().requires_grad_() for t in (x.new_zeros(*lead, 32), *ws, *bs)]
        y = kernel.mlp_packed(*none)
        assert y.shape == (*lead, 32)
        for t, g in zip(none, torch.autograd.grad(y, none, torch.zeros_like(y))):
            assert g.shape == t.shape and not g.any()
    turned = [t.detach().t().contiguous().t().requires_grad_() for t in ws]
    y = kernel.mlp_packed(x, *turned, *bs)
    assert torch.autograd.grad(y, turned, gy)[0].shape == ws[0].shape


def test_mlp_under_autocast():
    x, ws, bs, gy = _mlp_case(F32, (20,), 32, 64, 32, True)
    leaves = [t.detach().requires_grad_() for t in (x, *ws, *bs)]
    low = [t.detach().to(BF16).requires_grad_() for t in (x, *ws, *bs)]
    with torch.autocast("cuda", torch.bfloat16):
        y = kernel.mlp_packed(*leaves)
    want = kernel.mlp_packed(*low)
    assert y.dtype == BF16 and torch.equal(y, want)
    for a, b in zip(torch.autograd.grad(y, leaves, gy.to(BF16)), torch.autograd.grad(want, low, gy.to(BF16))):
        assert a.dtype == F32 and torch.equal(a, b.float())


def test_mlp_keeps_8_bits():
    """What the graph of the (C, 4 C) MLP holds: 5 C bytes and their exponents a row
    beside the result."""
    R, C = 4096, 256
    x, ws, _, _ = _mlp_case(BF16, (R,), C, 4 * C, C, False)
    leaves = [t.detach().requires_grad_() for t in (x, *ws)]
    kernel.mlp_packed(*leaves).sum().backward()              # workspaces of the products
    torch.cuda.synchronize()
    before = in_use()
    y = kernel.mlp_packed(*leaves)
    assert in_use() - before <= y.numel() * 2 + R * 5 * C * (1 + 1 / 32) + 8192


def test_mlp_is_differentiated_once():
    x, ws, bs, gy = _mlp_case(F32, (20,), 32, 64, 32, True)
    x.requires_grad_()
    (g,) = torch.autograd.grad(kernel.mlp_packed(x, *ws).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice|once_differentiable"):
        g.sum().backward()


def test_refusals():
    x = rnd(4, 32, seed=1)
    for call in (lambda t: kernel.pack_activation(t), lambda t: kernel.gelu_packed(t)):
        with pytest.raises(NotImplementedError, match="unsupported dtype"):
            call(x.double())
        with pytest.raises(NotImplementedError, match="unsupported dtype"):
            call(x.long())
        with pytest.raises(ValueError, match="at least one channel"):
            call(x[:, :0])
        with pytest.raises(ValueError, match="at least one channel"):
            call(x[0, 0])
    with pytest.raises(NotImplementedError, match="no backward"):
        kernel.pack_activation(x.clone().requires_grad_())
    p = kernel.pack_activation(x)
    for bad in (p._replace(exp=p.exp[:2]), p._replace(q=p.q.short()), p._replace(q=p.q[:, :31].contiguous(), exp=p.exp[:, :0]),
                p._replace(q=p.q[:, ::2])):
        with pytest.raises((ValueError, NotImplementedError)):
            kernel.unpack_activation(bad)
    assert math.isfinite(float(kernel.unpack_activation(p).sum()))
