"""Token log probabilities, entropy, top alternatives and gradients against
float64."""
import math

import pytest
import torch

import kernel
from decode_cases import HALF_STEP, logprob_reference

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(R, V, dtype=BF16, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, V, generator=g) * std).to(dtype)
    t = torch.randint(0, V, (R,), generator=g)
    return x, t


def _tol(ref, scale_of):
    """fp32 bound of a log probability: x' = x scale log2 e carries the
    rounding of scale log2 e (2^-24 relative, up to the spread of the row's
    exponents), exp2 / log2 one step each and the sum of e at most a few ten
    steps (pairwise over threads, each thread a few hundred terms in the worst
    case): 2^-17 of max(1, |value|, log V) is above all of these."""
    return 2.0 ** -17 * torch.clamp(ref.abs(), min=scale_of)


def _check(x, t, top=0, entropy=False, scale=1.0, **kw):
    r = kernel.token_logprobs(x.cuda(), t.cuda(), top=top, entropy=entropy, scale=scale, **kw)
    logp, ent, idx, tlp, _ = logprob_reference(x, t, top, scale)
    base = max(1.0, math.log(x.size(1)))
    assert r.logp.dtype == FP32
    same_nan = torch.isnan(r.logp.cpu()) == torch.isnan(logp)
    assert bool(same_nan.all())
    ok = torch.isfinite(logp)
    err = (r.logp.double().cpu() - logp).abs()
    assert bool((err <= _tol(logp, base))[ok].all()), float(err[ok].max())
    assert torch.equal(r.logp.cpu()[~ok].nan_to_num(nan=0.0), logp[~ok].float().nan_to_num(nan=0.0))
    if entropy:
        assert bool(((r.entropy.double().cpu() - ent).abs() <= _tol(ent, base)).all())
    else:
        assert r.entropy is None
    if top:
        assert torch.equal(r.top_index.cpu(), idx)
        fin = torch.isfinite(tlp)
        assert bool(((r.top_logp.double().cpu() - tlp).abs() <= _tol(tlp, base))[fin].all())
    else:
        assert r.top_index is None and r.top_logp is None
    return r


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (3, 65), (7, 513), (2, 2047), (2, 2049),
                                 (3, 10007), (1, 50257), (600, 1000), (600, 4097), (2, 151936)])
def test_sizes(R, V, dtype):
    x, t = _inputs(R, V, dtype, seed=V)
    _check(x, t)
    _check(x, t, top=min(V, 5), entropy=True, scale=0.7)


@pytest.mark.parametrize("top", [1, 2, 17, 31, 32])
@pytest.mark.parametrize("R,V", [(3, 32), (2, 40), (3, 300), (2, 5000), (600, 9001), (2, 60000)])
def test_top(R, V, top):
    x, t = _inputs(R, V, seed=top + V)
    _check(x, t, top=top)


@pytest.mark.parametrize("V", [40, 3000, 60001])
def test_ties_go_to_the_lower_index(V):
    for x in (torch.zeros(2, V), -torch.zeros(2, V), torch.full((2, V), -3.0), (torch.arange(V) % 3).float().expand(2, V)):
        x = x.contiguous().to(BF16)
        x[1, ::2] *= -1.0                    # -0.0 next to 0.0 ties as well
        _check(x, torch.zeros(2, dtype=torch.long), top=20, entropy=True)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_sorted_rows(dtype):
    """Ascending and descending rows, and rows whose largest elements sit in
    one thread's pieces (more candidates than the collection holds)."""
    V = 60000
    up = torch.linspace(-8, 8, V)
    x = torch.stack([up, up.flip(0), torch.zeros(V)])
    n = 16 // (2 if dtype == BF16 else 4)
    for nt in (64, 256, 512, 1024):
        piece = torch.arange(V) // n
        x = torch.cat([x, ((piece % nt < 20).float() * 4 + up * 0.01)[None]])
    # many rows of one segment each, and few rows in several
    for rows in (x, x.repeat(90, 1)):
        _check(rows.to(dtype), torch.zeros(rows.size(0), dtype=torch.long), top=20)


def test_every_element_a_candidate():
    """20 threads' pieces all hold values above everything else."""
    V, nt, n = 150000, 256, 8
    piece = torch.arange(V) // n
    x = torch.where(piece % nt < 20, 5.0 + (torch.arange(V) % 97) / 64.0, torch.zeros(V))
    x = x.to(BF16)[None].repeat(600, 1)
    _check(x, torch.zeros(600, dtype=torch.long), top=20)


@pytest.mark.parametrize("R,V,nt", [(600, 4000, 64), (100, 60000, 512), (3, 160000, 256), (600, 30000, 256)])
def test_candidates_of_every_block_size(R, V, nt):
    """The same in the one-wave, 512-thread and segmented forms, and with all
    large values in one thread's pieces."""
    piece = torch.arange(V) // 8
    many = torch.where(piece % nt < 20, 5.0 + (torch.arange(V) % 97) / 64.0, torch.zeros(V))
    one = torch.where(piece % nt == 3, 5.0 - (torch.arange(V) % 1009) / 512.0, torch.zeros(V))
    x = torch.stack([many, one, many.flip(0)]).to(BF16)
    x = x.repeat((R + 2) // 3, 1)[:R].contiguous()
    _check(x, torch.zeros(R, dtype=torch.long), top=20, entropy=True)


@pytest.mark.parametrize("V", [50, 5000, 40000])
def test_masked_rows(V):
    """-inf entries, the type's lowest value, fewer finite entries than top."""
    x, t = _inputs(4, V, BF16, seed=1)
    x[0, 3:] = -float("inf")
    x[1, :-1] = torch.finfo(BF16).min
    x[2, V // 2:] = -float("inf")
    t[:] = torch.tensor([1, V - 1, 0, 2])
    _check(x, t, top=8, entropy=True)
    t[2] = V - 1                             # a masked token: -inf
    r = kernel.token_logprobs(x.cuda(), t.cuda())
    assert float(r.logp[2]) == -float("inf")


@pytest.mark.parametrize("V", [50, 5000, 40000])
def test_rows_without_a_distribution(V):
    x, t = _inputs(4, V, BF16, seed=2)
    x[0] = -float("inf")
    x[1, V // 3] = float("nan")
    x[2, V // 5] = float("inf")
    r = kernel.token_logprobs(x.cuda(), t.cuda(), top=3, entropy=True)
    assert torch.isnan(r.logp[:3]).all() and torch.isnan(r.entropy[:3]).all() and torch.isnan(r.top_logp[:2]).all()
    assert ((r.top_index >= 0) & (r.top_index < V)).all()
    assert torch.isfinite(r.logp[3]) and torch.isfinite(r.top_logp[3]).all()


def test_ignored_and_outside_tokens():
    x, t = _inputs(5, 1000, seed=3)
    t[:] = torch.tensor([-100, 5, 1000, -1, 999])
    r = _check(x, t)
    assert float(r.logp[0]) == 0.0 and torch.isnan(r.logp[2:4]).all()
    r = kernel.token_logprobs(x.cuda(), t.cuda(), ignore_index=5)
    assert float(r.logp[1]) == 0.0 and torch.isnan(r.logp[0])


def test_leading_dims_and_int32():
    x, t = _inputs(6, 777, seed=4)
    a = kernel.token_logprobs(x.cuda(), t.cuda(), top=2, entropy=True)
    b = kernel.token_logprobs(x.view(2, 3, 777).cuda(), t.view(2, 3).int().cuda(), top=2, entropy=True)
    assert b.logp.shape == (2, 3) and b.top_index.shape == (2, 3, 2)
    assert torch.equal(a.logp, b.logp.view(-1)) and torch.equal(a.top_index, b.top_index.view(6, 2))
    s = kernel.token_logprobs(x[0].cuda(), t[0].cuda())
    assert s.logp.shape == () and torch.equal(s.logp, a.logp[0])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_rows(dtype, offset):
    x, t = _inputs(5, 1001, dtype, seed=5)
    buf = torch.full((5, 1007), float("nan"), dtype=dtype, device="cuda")
    view = buf[:, offset:offset + 1001]
    view.copy_(x)
    tt = torch.stack([t, t * 0 - 7], 1).cuda()[:, 0]
    r = kernel.token_logprobs(view, tt, top=4, entropy=True)
    want = kernel.token_logprobs(x.cuda(), t.cuda(), top=4, entropy=True)
    assert torch.equal(r.top_index, want.top_index)
    # another alignment changes which thread sums what: a few steps
    assert bool(((r.logp - want.logp).abs() <= 2.0 ** -18 * 8).all())
    col = x.t().contiguous().cuda().t()      # columns with a stride: copied
    assert torch.equal(kernel.token_logprobs(col, t.cuda()).logp, kernel.token_logprobs(x.cuda(), t.cuda()).logp)


def test_no_rows():
    r = kernel.token_logprobs(torch.zeros(0, 10, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), top=2,
                              entropy=True)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2)


# ---- gradients ----------------------------------------------------------------

def _grad_reference(x, t, g, ge, scale, ignore=-100):
    xd = x.double() * scale
    lq = xd - torch.logsumexp(xd, -1, keepdim=True)
    p = lq.exp()
    H = -(p * lq.clamp(min=-1e30)).sum(-1, keepdim=True)
    on = (t != ignore).double()
    d = -(g.double() * on)[:, None] * p
    d[torch.arange(len(t)), t.clamp(min=0)] += g.double() * on
    if ge is not None:
        d = d - ge.double()[:, None] * p * (lq.clamp(min=-1e30) + H)
    return d * scale


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("R,V", [(1, 1), (2, 9), (5, 513), (3, 8191), (2, 8193), (4, 50257), (700, 1000)])
@pytest.mark.parametrize("ent", [False, True])
def test_gradient(R, V, dtype, ent):
    x, t = _inputs(R, V, dtype, seed=R + V)
    if R > 2:
        t[1] = -100
    g = torch.linspace(-1.5, 1.0, R)
    ge = torch.linspace(0.7, -0.4, R) if ent else None
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda(), entropy=ent, scale=0.8, top=1)
    outs, gs = ([r.logp, r.entropy], [g.cuda(), ge.cuda()]) if ent else ([r.logp], [g.cuda()])
    (dx,) = torch.autograd.grad(outs, xg, gs)
    want = _grad_reference(x, t, g, ge, 0.8)
    assert dx.dtype == dtype and dx.shape == x.shape
    # p carries the exponent's fp32 error (2^-18 relative at exponents of 30);
    # with the entropy's it is multiplied by |log p + H| <= 40, and g (1 - p)
    # is a difference of terms of size <= 2; plus the output's rounding and,
    # in fp16, its smallest step.  Each element takes three more fp32 roundings
    # of its own size, 2^-24 relative each: the sum with g, the product with
    # scale, and scale itself (0.8 in fp32 against 0.8)
    p = torch.softmax(x.double() * 0.8, -1)
    tol = (HALF_STEP[dtype] + 3 * 2.0 ** -24) * want.abs() + 2.0 ** -16 * (p * (40.0 if ent else 2.0)) + 2.0 ** -22 * (p > 0.01)
    tol = tol + {FP16: 2.0 ** -25, BF16: 0.0, FP32: 0.0}[dtype] + 1e-37
    err = (dx.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if R > 2 and not ent:
        assert (dx[1] == 0).all()


def test_gradient_against_differences():
    """Directional derivative of a weighted sum of logp and entropy, by central
    differences of the float32 operator: step 2^-6 leaves a third-order term
    of about step^2 / 6 = 4e-5 of the gradient's size and fp32 noise of
    2^-20 / 2^-6 = 6e-5."""
    x, t = _inputs(4, 400, FP32, seed=6)
    g = torch.Generator().manual_seed(8)
    d = torch.randn(4, 400, generator=g).cuda()
    a, b = torch.rand(4, generator=g).cuda(), torch.rand(4, generator=g).cuda()

    def f(v):
        r = kernel.token_logprobs(v, t.cuda(), entropy=True, scale=1.3)
        return (a * r.logp + b * r.entropy)

    xg = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(f(xg).sum(), xg)
    h = 2.0 ** -6
    num = ((f(x.cuda() + h * d) - f(x.cuda() - h * d)).double() / (2 * h)).cpu()
    ana = (dx * d).double().sum(-1).cpu()
    assert bool(((num - ana).abs() <= 2e-3 * (1 + ana.abs())).all())


def test_gradient_layouts():
    """Broadcast upstream gradients, strided logits, leading dims."""
    x, t = _inputs(6, 1001, seed=7)
    ref = _grad_reference(x, t, torch.full((6,), -1 / 6), None, 1.0)
    buf = torch.zeros(6, 1010, dtype=BF16, device="cuda")
    buf[:, 3:1004] = x.cuda()
    buf.requires_grad_()
    loss = -kernel.token_logprobs(buf[:, 3:1004].unflatten(0, (2, 3)), t.view(2, 3).cuda()).logp.mean()
    loss.backward()
    got = buf.grad.double().cpu()
    assert (got[:, :3] == 0).all() and (got[:, 1004:] == 0).all()
    assert bool(((got[:, 3:1004] - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -16).all())


def test_padding_rows_have_zero_gradient_whatever_they_hold():
    x, t = _inputs(3, 5000, seed=9)
    x[1] = float("nan")
    t[1] = -100
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda())
    assert float(r.logp[1].detach()) == 0.0
    r.logp.sum().backward()
    assert (xg.grad[1] == 0).all() and torch.isfinite(xg.grad).all()


def test_padding_rows_of_an_entropy_term():
    x, t = _inputs(3, 700, seed=12)
    x[1] = float("nan")
    t[1] = -100
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda(), entropy=True)
    keep = torch.tensor([0, 2]).cuda()
    (r.logp[keep].sum() + r.entropy[keep].sum()).backward()
    assert (xg.grad[1] == 0).all() and torch.isfinite(xg.grad).all()


def test_entropy_alone():
    x, t = _inputs(4, 900, FP32, seed=13)
    ge = torch.linspace(-1, 1, 4)
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda(), entropy=True)
    (dx,) = torch.autograd.grad(r.entropy, xg, ge.cuda())
    want = _grad_reference(x, t, torch.zeros(4), ge, 1.0)
    p = torch.softmax(x.double(), -1)
    assert bool(((dx.double().cpu() - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -16 * 40 * p + 1e-37).all())


def test_second_derivatives_are_refused():
    x, t = _inputs(2, 50, FP32, seed=14)
    xg = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(kernel.token_logprobs(xg, t.cuda()).logp.sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), xg)


def test_expanded_rows_and_another_stream():
    x, t = _inputs(1, 3000, seed=15)
    one = kernel.token_logprobs(x.cuda(), t.cuda(), top=3)
    many = kernel.token_logprobs(x.cuda().expand(5, -1), t.cuda().expand(5), top=3)
    assert all(torch.equal(a.expand(5, *a.shape[1:]), b) for a, b in zip(one[:1] + one[2:], many[:1] + many[2:]))
    side = torch.cuda.Stream()
    xd, td = x.cuda(), t.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kernel.token_logprobs(xd, td, top=3)
    side.synchronize()
    assert torch.equal(other.logp, one.logp) and torch.equal(other.top_index, one.top_index)


def test_masked_entries_have_zero_gradient():
    x, t = _inputs(2, 600, FP32, seed=10)
    x[0, 100:] = -float("inf")
    t[0] = 7
    xg = x.cuda().requires_grad_()
    r = kernel.token_logprobs(xg, t.cuda(), entropy=True)
    (r.logp.sum() + r.entropy.sum()).backward()
    assert (xg.grad[0, 100:] == 0).all() and torch.isfinite(xg.grad).all()


def test_same_answer_twice():
    x, t = _inputs(3, 60000, seed=11)
    a = kernel.token_logprobs(x.cuda(), t.cuda(), top=20, entropy=True)
    b = kernel.token_logprobs(x.cuda(), t.cuda(), top=20, entropy=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
