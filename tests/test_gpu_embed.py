"""kernel.embed_tokens against its definition in 64 bits: the lookup is one product
and one rounding, so equal to torch's; a gradient row is a float32 sum of n terms,
off by at most (n - 1) U of the sum of their magnitudes, one product and one
rounding."""
import pytest
import torch

import kernel
from kernel import _ext
from train_cases import BF16, DEV, F16, F32, HALF, LEAST, U, close, rnd

pytestmark = pytest.mark.gpu


def _tokens(N, V, seed, skew=1.0, dtype=torch.long):
    g = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.empty(N, device=DEV, dtype=torch.float64).uniform_(0, 1, generator=g)
    return (u ** skew * V).long().clamp(max=V - 1).to(dtype)


def _check(tokens, w, dy, scale, ignore=-100, dtype=None):
    w = w.detach().requires_grad_()
    y = kernel.embed_tokens(tokens, w, scale=scale, ignore_index=ignore, dtype=dtype)
    V, C = w.shape
    out_t = dtype or w.dtype
    assert y.shape == (*tokens.shape, C) and y.dtype == out_t
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < V) & (flat != ignore)
    want = (w.detach()[flat.clamp(0, V - 1)].float() * scale).to(out_t)
    want[~ok] = float("nan")
    want[flat == ignore] = 0
    assert torch.equal(y.detach().reshape(-1, C).nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
    (dw,) = torch.autograd.grad(y, w, dy)
    assert dw.dtype == w.dtype and dw.shape == w.shape and dw.is_contiguous()
    at, g = flat[ok], dy.reshape(-1, C)[ok].double()
    ref = torch.zeros(V, C, dtype=torch.float64, device=DEV).index_add_(0, at, g) * scale
    mag = torch.zeros_like(ref).index_add_(0, at, g.abs()) * abs(scale)
    n = torch.bincount(at, minlength=V).double()[:, None]
    close(dw, ref, (n + 1) * U * mag + HALF[w.dtype] * ref.abs() * (1 + 1e-6) + (LEAST[w.dtype] if n.any() else 0), "dw")
    absent = n[:, 0] == 0
    assert not dw[absent].any()
    return dw


@pytest.mark.parametrize("wt,yt", [(BF16, BF16), (F16, F16), (F32, F32), (F32, BF16), (F32, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("N,V,C", [(1, 1, 1), (2, 3, 8), (65, 300, 33), (1000, 70, 96), (1023, 5000, 257)])
def test_types_and_sizes(wt, yt, N, V, C):
    t = _tokens(N, V, N, skew=2.0)
    if N > 2:
        t[::7] = -100
    _check(t, rnd(V, C, seed=1, dtype=wt), rnd(N, C, seed=2, dtype=yt), 1.0 if C % 2 else 3.3, dtype=yt)


@pytest.mark.parametrize("N", [15, 16, 17, 63, 64, 65, 255, 256, 257, 1023, 8191, 8192, 8193, 10240, 16384, 16385, 40000])
@pytest.mark.parametrize("V", [2, 511, 512, 40000, 262143, 300000])
def test_sorting(N, V):
    """Few tokens, one to three passes, one tile and several, chunks of 16 and 32 positions, words
    of one position and of thousands."""
    t = _tokens(N, V, N + V, skew=3.0)
    t[5::11] = -100
    _check(t, rnd(V, 5, seed=3), rnd(N, 5, seed=4), 1.0)


@pytest.mark.parametrize("N", [1, 16, 40, 64, 65, 256, 257, 9000, 140001])
@pytest.mark.parametrize("word", [0, 96])
def test_one_word(N, word):
    t = torch.full((N,), word, device=DEV)
    _check(t, rnd(97, 40, seed=5), rnd(N, 40, seed=6), 0.5)


def test_many_tokens():
    """Longer chunks, tens of tiles; words that cross any number of chunks."""
    t = _tokens(200003, 1000, 8, skew=6.0)
    t[::3] = 17
    _check(t, rnd(1000, 24, seed=7), rnd(200003, 24, seed=8, dtype=F32), 1.0)


@pytest.mark.parametrize("V", [300, 70000])
def test_very_many_tokens(V):
    """More tiles than a workgroup adds up by itself; an odd number of them."""
    N = 2048 * 150 + 77
    t = _tokens(N, V, 8, skew=5.0)
    t[::5] = 3
    t[1::50] = -100
    _check(t, rnd(V, 3, seed=7), rnd(N, 3, seed=8, dtype=F32), 1.0)


@pytest.mark.parametrize("tt", [torch.long, torch.int32])
def test_tokens_out_of_range(tt):
    t = _tokens(100, 50, 9, dtype=tt)
    t[3], t[4], t[5], t[6], t[7] = -1, 50, -100, torch.iinfo(tt).max, torch.iinfo(tt).min
    _check(t, rnd(50, 48, seed=10, dtype=BF16), rnd(100, 48, seed=11, dtype=BF16), 2.0)
    # the ignored token may be a word, or nothing in reach
    _check(t, rnd(50, 48, seed=10), rnd(100, 48, seed=11), 2.0, ignore=7)


def test_all_ignored_and_empty():
    w = rnd(50, 48, seed=10, dtype=BF16)
    _check(torch.full((33,), -100, device=DEV), w, rnd(33, 48, seed=1, dtype=BF16), 1.0)
    _check(torch.full((33,), 1000, device=DEV), w, rnd(33, 48, seed=1, dtype=BF16), 1.0)
    dw = _check(torch.empty(0, dtype=torch.long, device=DEV), w, rnd(0, 48, seed=1, dtype=BF16), 1.0)
    assert not dw.any()
    _check(torch.empty(0, 7, dtype=torch.long, device=DEV), w, torch.zeros(0, 7, 48, device=DEV, dtype=BF16), 1.0)


def test_layouts():
    """Tokens, gradients and weights of other strides than the usual."""
    t = _tokens(60, 50, 12).view(3, 20)
    w, dy = rnd(50, 40, seed=13), rnd(3, 20, 40, seed=14)
    want = _check(t, w, dy, 1.0)
    base = torch.zeros(20, 6, dtype=torch.long, device=DEV)
    base[:, ::2] = t.t()
    for tokens in (base[:, ::2].t(), t.t().contiguous().t(), t.int()):
        assert torch.equal(_check(tokens, w, dy, 1.0), want)
    wide = torch.zeros(3, 20, 81, device=DEV)
    wide[..., 1:41] = dy
    for g in (wide[..., 1:41], dy.transpose(0, 2).contiguous().transpose(0, 2), dy.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(_check(t, w, g, 1.0), want)
    _check(t, w, torch.ones((), device=DEV).expand(3, 20, 40), 1.0)
    ww = torch.zeros(50, 83, device=DEV)
    ww[:, 3:43] = w
    for weight in (ww[:, 3:43], w.t().contiguous().t()):
        y = kernel.embed_tokens(t, weight)
        assert torch.equal(y, w[t])
        leaf = weight.detach().requires_grad_()
        (dw,) = torch.autograd.grad(kernel.embed_tokens(t, leaf), leaf, dy)
        assert torch.equal(dw, want)


def test_one_row_of_tokens():
    t = torch.tensor(3, device=DEV)                      # no dimension at all
    w = rnd(5, 8, seed=1)
    assert torch.equal(kernel.embed_tokens(t, w), w[3])


def test_same_bits_every_time():
    t, w, dy = _tokens(20000, 700, 20, skew=4.0), rnd(700, 100, seed=21, dtype=BF16), rnd(20000, 100, seed=22, dtype=BF16)
    first = _check(t, w, dy, 1.7)
    for _ in range(4):
        assert torch.equal(_check(t, w, dy, 1.7), first)


def test_rows_past_32_bits():
    """An embedding of more than 2^32 elements: its last rows, and their gradient."""
    V, C = (1 << 21) + 5, 2049
    w = torch.zeros(V, C, device=DEV, dtype=BF16)
    w[-1], w[0] = 3, 1
    w.requires_grad_()
    t = torch.tensor([V - 1, 0, V - 1, V], device=DEV)
    y = kernel.embed_tokens(t, w)
    assert (y[0] == 3).all() and (y[1] == 1).all() and y[3].isnan().all()
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert (dw[-1] == 2).all() and (dw[0] == 1).all()
    assert not dw[1:-1].any()


def test_against_differences():
    """The lookup is linear: differences of any length are its gradient, to the
    rounding of the two arguments, of their products, and of a gradient's sum of at
    most 65 / 30 x 4 terms: 16 U of the magnitudes."""
    t, w, dy, v = _tokens(65, 30, 1), rnd(30, 40, seed=2), rnd(65, 40, seed=3), rnd(30, 40, seed=4)
    leaf = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(kernel.embed_tokens(t, leaf, scale=1.5), leaf, dy)
    f = lambda a: (kernel.embed_tokens(t, a, scale=1.5).double() * dy.double()).sum()   # noqa: E731
    want, got = (f(w + v) - f(w - v)) / 2, (dw.double() * v.double()).sum()
    assert abs(want - got) <= 16 * U * (kernel.embed_tokens(t, w.abs() + v.abs(), scale=1.5).double() * dy.abs()).sum()


def test_no_second_derivative():
    w = rnd(5, 8, seed=1).requires_grad_()
    y = kernel.embed_tokens(torch.tensor([1, 2], device=DEV), w)
    (g,) = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="twice differentiating"):
        g.sum().backward()


def test_refusals():
    w, t = rnd(5, 8, seed=1), torch.tensor([1, 2], device=DEV)
    with pytest.raises(ValueError, match="tokens must be int32 or int64"):
        kernel.embed_tokens(t.float(), w)
    with pytest.raises(NotImplementedError, match="beside fp16"):
        kernel.embed_tokens(t, w.bfloat16(), dtype=F16)
    with pytest.raises(ValueError, match="weight must be"):
        kernel.embed_tokens(t, w[0])
    with pytest.raises(ValueError, match="expected cuda"):
        kernel.embed_tokens(t.cpu(), w)
    with pytest.raises(NotImplementedError, match="unsupported dtype"):
        kernel.embed_tokens(t, w.double())
    assert _ext.lib().saf_version()
