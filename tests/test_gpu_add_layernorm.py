"""kernel.add_layernorm against its definition in 64 bits, forward and backward,
with the float32 error bounds of train_cases.norm_exact and one rounding of each
result."""
import math

import pytest
import torch

import kernel
from train_cases import BF16, DEV, F16, F32, HALF, LEAST, U, close, norm_exact, rnd

pytestmark = pytest.mark.gpu

TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (F32, F16)]


def _check(x, delta, w, b, dy, dr, eps=1e-5, dtype=None):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, delta, w, b)]
    r, y = kernel.add_layernorm(*leaves, eps=eps, dtype=dtype)
    C = x.size(-1)
    f = lambda t: None if t is None else t.reshape(-1, C)   # noqa: E731
    want, tol = norm_exact(f(x), f(delta), w, b, eps, f(dy), f(dr))
    assert r.shape == y.shape == x.shape
    assert torch.equal(f(r.detach()).nan_to_num(nan=7.0), want[0].nan_to_num(nan=7.0))
    if delta is None:
        assert r is leaves[0]
    yt = dy.dtype
    assert y.dtype == yt
    round_ = lambda t, ref: HALF[t] * ref.abs() * (1 + 1e-6) + LEAST[t]   # noqa: E731
    close(f(y.detach()), want[1], tol[1] + round_(yt, want[1]), "y")
    heads, seeds = ((y,), (dy,)) if dr is None else ((r, y), (dr, dy))
    used = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("x", "delta", "w", "b"), leaves) if t is not None],
                     torch.autograd.grad(heads, used, seeds)))
    close(f(grads["x"]), want[2], tol[2] + round_(x.dtype, want[2]), "dx")
    if delta is not None:
        close(f(grads["delta"]), want[2], tol[2] + round_(delta.dtype, want[2]), "ddelta")
    close(grads["w"], want[3], tol[3] + round_(w.dtype, want[3]), "dw")
    if b is not None:
        close(grads["b"], want[4], tol[4] + round_(b.dtype, want[4]), "db")
    for n, t in zip(("x", "delta", "w", "b"), leaves):
        if t is not None:
            assert grads[n].dtype == t.dtype and grads[n].shape == t.shape
    return [r.detach(), y.detach(), *grads.values()]


def _case(R, C, xt, yt, wt, delta=True, bias=True, seed=0):
    return dict(x=rnd(R, C, seed=seed, dtype=xt) * 2 + 0.5, delta=rnd(R, C, seed=seed + 1, dtype=yt) if delta else None,
                w=1 + rnd(C, seed=seed + 2, std=0.3, dtype=wt), b=rnd(C, seed=seed + 3, dtype=wt) if bias else None,
                dy=rnd(R, C, seed=seed + 4, dtype=yt), dr=rnd(R, C, seed=seed + 5, dtype=xt) if delta else None)


@pytest.mark.parametrize("xt,yt", TYPES)
@pytest.mark.parametrize("C", [1, 7, 8, 33, 64, 65, 128, 129, 256, 257, 511, 768, 1000, 1024, 1025, 1536, 2047, 2048, 2049, 4100, 6144, 8191])
def test_widths_and_types(xt, yt, C):
    """Every layout of a row: eight lanes to four waves, 1 to 4 chunks a thread."""
    c = _case(37, C, xt, yt, yt if C % 2 else F32, delta=C % 3 != 0, bias=C % 4 != 0, seed=C)
    _check(**c, dtype=yt)


def _among_nans(t, gap):
    """t's values as rows gap apart, with NaNs between and around them."""
    R, C = t.shape
    buf = torch.full((R + 2, C + gap), math.nan, device=DEV, dtype=t.dtype)
    view = buf[1:-1, gap // 2:gap // 2 + C]
    view.copy_(t)
    return view


@pytest.mark.parametrize("xt,yt", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("chunks", [8, 9, 20, 40, 80, 100, 150, 200, 256, 300, 450, 700, 900, 1100])
def test_last_chunks(xt, yt, chunks):
    """Every size of a last chunk in every layout, whole ones of the wider layouts too;
    nothing of what lies around a row gets into it."""
    for rest in range(8):
        c = _case(9, 8 * chunks + rest, xt, yt, xt, seed=chunks + rest)
        for k in ("x", "delta", "dy", "dr"):
            c[k] = _among_nans(c[k], 5 + rest)
        _check(**c, dtype=yt)


@pytest.mark.parametrize("C", [8193, 16384])
@pytest.mark.parametrize("xt,yt", [(BF16, BF16), (F32, F16)])
def test_widest(xt, yt, C):
    _check(**_case(5, C, xt, yt, F32, seed=C), dtype=yt)


@pytest.mark.parametrize("R", [1, 2, 4, 5, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 128, 129, 4095, 4096, 5001])
@pytest.mark.parametrize("C", [40, 100, 64, 1280, 2100])
def test_rows(R, C):
    """One workgroup, fewer rows than workgroups, and more: ragged last rounds."""
    _check(**_case(R, C, BF16, BF16, BF16, seed=R))


def test_no_rows():
    for C in (3, 64):
        for wt in (F32, BF16):
            out = _check(**_case(0, C, BF16, BF16, wt))
            assert not out[-1].any() and not out[-2].any()
    x = torch.zeros(2, 0, 64, device=DEV)
    r, y = kernel.add_layernorm(x, x, torch.ones(64, device=DEV))
    assert r.shape == y.shape == x.shape


def test_shapes():
    c = _case(24, 40, F32, F32, F32)
    want = _check(**c)
    for shape in ((2, 3, 4, 40), (24, 1, 40)):
        d = {k: v if v is None or k in "wb" else v.view(shape) for k, v in c.items()}
        for a, b in zip(_check(**d), want):
            assert torch.equal(a.reshape(b.shape), b)
    one = {k: v if v is None or k in "wb" else v[:1] for k, v in c.items()}
    want = _check(**one)
    for a, b in zip(_check(**{k: v if v is None or k in "wb" else v[0] for k, v in one.items()}), want):
        assert torch.equal(a.reshape(b.shape), b)


@pytest.mark.parametrize("C", [40, 41, 768])
def test_layouts(C):
    """Row strides, odd offsets, transposed and broadcast operands."""
    c = _case(30, C, BF16, BF16, BF16, seed=3)
    want = _check(**c)

    def wide(t):
        big = torch.zeros(30, C + 5, device=DEV, dtype=t.dtype)
        big[:, 3:3 + C] = t
        return big[:, 3:3 + C]

    for change in (wide, lambda t: t.t().contiguous().t()):
        d = {k: v if k in "wb" else change(v) for k, v in c.items()}
        for a, b in zip(_check(**d), want):
            assert torch.equal(a, b)
    every = torch.zeros(2 * C, device=DEV, dtype=BF16)
    every[::2] = c["w"]
    for a, b in zip(_check(**dict(c, w=every[::2])), want):
        assert torch.equal(a, b)
    _check(**dict(c, dy=torch.ones((), device=DEV, dtype=BF16).expand(30, C), dr=c["dr"][:1].expand(30, C)))


def test_numbers_at_the_edges():
    """Rows without variance, far from zero, infinite, NaN: each keeps to itself;
    channels of the weight gradients that meet a NaN are NaN, as the formula says."""
    c = _case(9, 100, F32, F32, F32, delta=False, seed=4)
    c["x"][0] = 0
    c["x"][1] = 5
    c["x"][2] = 1e6 + rnd(100, seed=9)
    c["x"][3] *= 1e-20
    c["x"][4] *= 1e15
    _check(**c)
    c["x"][5, 7], c["x"][6, 8], c["x"][7, 9] = float("nan"), float("inf"), float("-inf")
    x = c["x"].requires_grad_()
    _, y = kernel.add_layernorm(x, None, c["w"], c["b"])
    (dx,) = torch.autograd.grad(y, x, c["dy"])
    assert y[5:8].isnan().all() and dx[5:8].isnan().all()
    assert y[:5].isfinite().all() and dx[:5].isfinite().all() and y[8].isfinite().all() and dx[8].isfinite().all()


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1.0])
def test_eps(eps):
    _check(**_case(10, 65, F32, F32, F32), eps=eps)


@pytest.mark.parametrize("xt,yt", TYPES)
def test_part_of_the_gradients(xt, yt):
    """Any inputs that need one, with either output used alone."""
    c = _case(50, 96, xt, yt, F32, seed=6)
    full = _check(**c, dtype=yt)
    names = ("x", "delta", "w", "b")
    for mask in range(1, 16):
        leaves = [c[n].detach().requires_grad_(bool(mask >> i & 1)) for i, n in enumerate(names)]
        r, y = kernel.add_layernorm(*leaves)
        got = torch.autograd.grad((r, y) if mask & 3 else (y,), [t for t in leaves if t.requires_grad],
                                  (c["dr"], c["dy"]) if mask & 3 else (c["dy"],))
        for g, i in zip(got, [i for i in range(4) if mask >> i & 1]):
            assert torch.equal(g, full[2 + i]), (mask, names[i])
    # y alone: no dr; r alone: its own gradient and nothing for w and b
    leaves = [c[n].detach().requires_grad_() for n in names]
    r, y = kernel.add_layernorm(*leaves)
    want = _check(**dict(c, dr=torch.zeros_like(c["dr"])), dtype=yt)
    got = torch.autograd.grad(y, leaves, c["dy"], retain_graph=True)
    for g, w in zip(got, want[2:]):
        assert torch.equal(g, w)
    got = torch.autograd.grad(r, leaves, c["dr"], allow_unused=True)
    assert torch.equal(got[0], c["dr"]) and torch.equal(got[1], c["dr"].to(yt)) and got[2] is None and got[3] is None


def test_gradients_add_up():
    """backward() into leaves that already hold a gradient, and one tensor as x
    and as delta."""
    c = _case(20, 64, F32, F32, F32, seed=8)
    x, w = c["x"].requires_grad_(), c["w"].requires_grad_()
    for _ in range(2):
        r, y = kernel.add_layernorm(x, x, w)
        (y * c["dy"]).sum().backward()
    want, tol = norm_exact(c["x"].detach(), c["x"].detach(), w.detach(), None, 1e-5, c["dy"])
    close(x.grad, 4 * want[2], 4 * tol[2] + 8 * U * want[2].abs(), "dx")
    close(w.grad, 2 * want[3], 2 * tol[3] + 4 * U * want[3].abs(), "dw")


def test_same_bits_every_time():
    c = _case(3000, 300, BF16, BF16, F32, seed=9)
    first = _check(**c)
    for _ in range(3):
        for a, b in zip(_check(**c), first):
            assert torch.equal(a, b)


def test_rows_past_32_bits():
    R, C = (1 << 18) + 3, 16384
    x = torch.zeros(R, C, device=DEV, dtype=BF16)
    x[-1] = rnd(C, seed=1)
    w = torch.ones(C, device=DEV)
    r, y = kernel.add_layernorm(x, None, w)
    assert torch.equal(y[-1], kernel.add_layernorm(x[-1].clone(), None, w)[1]) and not y[1].any()
    del r, y
    x.requires_grad_()
    _, y = kernel.add_layernorm(x[-2:], None, w)
    dy = rnd(2, C, seed=2, dtype=BF16)
    (g,) = torch.autograd.grad(y, x, dy)
    (want,) = torch.autograd.grad(kernel.add_layernorm(s := x[-2:].detach().clone().requires_grad_(), None, w)[1], s, dy)
    assert torch.equal(g[-2:], want)


def test_against_differences():
    """Central differences along a direction: their second-order error is bounded by
    h^2 / 6 of the third derivative, estimated from two lengths (Richardson), the
    float32 rounding of the values by their count."""
    c = _case(6, 50, F32, F32, F32, seed=11)
    dirs = {n: rnd(*c[n].shape, seed=20 + i) for i, n in enumerate(("x", "delta", "w", "b"))}
    leaves = {n: c[n].detach().requires_grad_() for n in dirs}
    r, y = kernel.add_layernorm(leaves["x"], leaves["delta"], leaves["w"], leaves["b"])
    got = torch.autograd.grad((r, y), list(leaves.values()), (c["dr"], c["dy"]))

    def f(h, n):
        a = {k: c[k] + (h * dirs[k] if k == n else 0) for k in dirs}
        r, y = kernel.add_layernorm(a["x"], a["delta"], a["w"], a["b"])
        return ((r.double() * c["dr"]).sum() + (y.double() * c["dy"]).sum()).item()

    noise = 64 * U * float(c["dy"].abs().sum() * 3 + c["dr"].abs().sum() * 4)
    for n, g in zip(dirs, got):
        d1, d2 = ((f(h, n) - f(-h, n)) / (2 * h) for h in (0.04, 0.02))
        assert abs((4 * d2 - d1) / 3 - (g.double() * dirs[n]).sum().item()) <= abs(d1 - d2) + noise / 0.02, n


def test_changed_inputs_are_noticed():
    c = _case(4, 32, F32, F32, F32)
    x = c["x"].requires_grad_()
    r, y = kernel.add_layernorm(x, c["delta"], c["w"])
    r.data_ptr()
    with torch.no_grad():
        r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_no_second_derivative():
    c = _case(4, 32, F32, F32, F32)
    x = c["x"].requires_grad_()
    _, y = kernel.add_layernorm(x, c["delta"], c["w"])
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice differentiating"):
        g.sum().backward()


def test_refusals():
    x, w = rnd(4, 32, seed=1), rnd(32, seed=2)
    with pytest.raises(ValueError, match="share a shape"):
        kernel.add_layernorm(x, x[:1], w)
    with pytest.raises(NotImplementedError, match="with float32 y"):
        kernel.add_layernorm(x.bfloat16(), None, w, dtype=F32)
    with pytest.raises(NotImplementedError, match="with float16 y"):
        kernel.add_layernorm(x.bfloat16(), x.half(), w)
    with pytest.raises(ValueError, match="delta"):
        kernel.add_layernorm(x, x, w, dtype=BF16)
    with pytest.raises(ValueError, match="weight must be"):
        kernel.add_layernorm(x, None, w[:31])
    with pytest.raises(ValueError, match="bias must be"):
        kernel.add_layernorm(x, None, w, w.half())
    with pytest.raises(NotImplementedError, match="C = 16385"):
        kernel.add_layernorm(torch.zeros(1, 16385, device=DEV), None, torch.zeros(16385, device=DEV))
    with pytest.raises(ValueError, match="expected cuda"):
        kernel.add_layernorm(x, None, w.cpu())
