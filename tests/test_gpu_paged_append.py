"""New tokens into a paged cache against float64: norm, rotation, pages, and
everything that must stay as it was."""
import pytest
import torch

import kernel
from decode_cases import HALF_STEP, append_reference

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _case(B=2, T=3, Uq=4, Uk=2, Hv=2, hd=64, rd=64, page=16, dtype=BF16, norm=True, starts=(0, 5), counts=None, seed=0,
          cs_dtype=FP32, cs_rows=None):
    g = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g).to(dtype)

    n_tab = max((s + T + page - 1) // page for s in starts)
    P = B * n_tab + 2
    table = torch.randperm(P, generator=g)[:B * n_tab].view(B, n_tab).int()
    top = cs_rows or max(starts) + T
    ang = torch.outer(torch.arange(top).double(), 10000.0 ** (-torch.arange(0, rd, 2).double() / rd)) if rd else None
    ang = torch.cat([ang, ang], -1) if rd else None
    y = randn(B, T, Uq + Uk + Hv, hd).transpose(1, 2)
    return dict(q=y[:, :Uq], k=y[:, Uq:Uq + Uk], v=y[:, Uq + Uk:], kc=randn(P, Uk, page, hd), vc=randn(P, Hv, page, hd),
                table=table, positions=torch.tensor(starts, dtype=torch.int32),
                counts=None if counts is None else torch.tensor(counts, dtype=torch.int32),
                cos=ang.cos().to(cs_dtype) if rd else None, sin=ang.sin().to(cs_dtype) if rd else None,
                qw=(1 + 0.1 * randn(hd).float()).to(dtype) if norm else None,
                kw=(1 + 0.1 * randn(hd).float()).to(dtype) if norm else None, page=page)


def _run(c, with_q=True):
    y = c["q"]
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    q = kernel.paged_append_(dev["k"], dev["v"], dev["kc"], dev["vc"], dev["table"], dev["positions"], dev["counts"],
                             q=dev["q"] if with_q else None, cos=dev["cos"], sin=dev["sin"], q_weight=dev["qw"],
                             k_weight=dev["kw"], eps=1e-5)
    assert torch.equal(dev["q"].cpu(), y)       # the inputs are only read
    return q, dev["kc"], dev["vc"]


def _check(c):
    q, kc, vc = _run(c)
    dt = c["vc"].dtype
    B, Hv, T, hd = c["v"].shape
    counts = [T] * B if c["counts"] is None else c["counts"].tolist()
    ek, ev = c["kc"].double(), c["vc"].clone()
    eq = torch.zeros(c["q"].shape, dtype=torch.float64)
    touched = torch.zeros(kc.shape[0], c["page"], dtype=torch.bool)
    for b in range(B):
        for t in range(counts[b]):
            s = int(c["positions"][b]) + t
            pg, sl = int(c["table"][b, s // c["page"]]), s % c["page"]
            eq[b, :, t] = append_reference(c["q"][b, :, t], c["qw"], 1e-5, c["cos"], c["sin"], s)
            ek[pg, :, sl] = append_reference(c["k"][b, :, t], c["kw"], 1e-5, c["cos"], c["sin"], s)
            ev[pg, :, sl] = c["v"][b, :, t]
            touched[pg, sl] = True
    assert torch.equal(vc.cpu(), ev)
    untouched = ~touched[:, None, :, None].expand(kc.shape)
    assert torch.equal(kc.cpu()[untouched], c["kc"][untouched])
    # one rounding of the result, and in fp32 before it the sum of squares
    # (hd 2^-24), rsqrt and four products (8 2^-24) of terms of size <= 8 (a
    # rotated pair of normal values times weights near 1)
    for got, want in ((q.cpu().double(), eq), (kc.cpu().double(), ek)):
        tol = HALF_STEP[dt] * want.abs() + (hd + 16) * 2.0 ** -24 * 8
        assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hd,rd", [(32, 32), (64, 64), (64, 16), (96, 96), (96, 48), (128, 128), (256, 64), (256, 256)])
@pytest.mark.parametrize("norm", [False, True])
def test_head_dims(hd, rd, dtype, norm):
    _check(_case(hd=hd, rd=rd, dtype=dtype, norm=norm, seed=hd + rd))


@pytest.mark.parametrize("T,starts,counts", [(1, (0, 31), None), (1, (15, 16), (1, 0)), (17, (0, 3), None),
                                             (40, (7, 0), (40, 13)), (5, (12, 30), (0, 9))])
def test_positions(T, starts, counts):
    if counts and max(counts) > T:
        counts = tuple(min(c, T) for c in counts)
    _check(_case(T=T, starts=starts, counts=counts, seed=T))


@pytest.mark.parametrize("Uq,Uk,Hv", [(1, 1, 1), (9, 9, 12), (14, 2, 2), (3, 3, 5)])
def test_heads(Uq, Uk, Hv):
    _check(_case(Uq=Uq, Uk=Uk, Hv=Hv, T=4, seed=Uq))


@pytest.mark.parametrize("cs_dtype", [FP32, BF16, FP16])
def test_rotary_cache_types(cs_dtype):
    _check(_case(cs_dtype=cs_dtype, seed=2))


def test_no_rotation():
    _check(_case(rd=0, seed=3))
    _check(_case(rd=0, norm=False, seed=4))


def test_counts_above_tokens_write_only_what_is_there():
    c = _case(T=3, seed=5)
    c["counts"] = torch.tensor([7, 3], dtype=torch.int32)
    q, kc, vc = _run(c)
    c["counts"] = None
    q2, kc2, vc2 = _run(c)
    assert torch.equal(q, q2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_no_live_heads():
    c = _case(seed=6)
    d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    assert kernel.paged_append_(None, d["v"], None, d["vc"], d["table"], d["positions"]) is None
    pg, sl = int(c["table"][1, 0]), 5
    assert torch.equal(d["vc"][pg, :, sl].cpu(), c["v"][1, :, 0])
    empty = d["q"][:, :0]
    q = kernel.paged_append_(empty, d["v"], None if False else d["kc"][:, :0], d["vc"], d["table"], d["positions"],
                             q=empty, cos=d["cos"], sin=d["sin"])
    assert q.shape == empty.shape


def test_without_q():
    c = _case(seed=7)
    q, kc, vc = _run(c, with_q=False)
    _, kc2, vc2 = _run(c)
    assert q is None and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_outside_positions_and_bad_pages():
    """Not written, NaN query rows, and nothing else changes."""
    c = _case(T=4, starts=(0, 5), seed=8)
    good = _run(c)
    c["positions"] = torch.tensor([-2, c["table"].size(1) * 16 - 2], dtype=torch.int32)
    q, kc, vc = _run(c)
    q = q.float().cpu()
    assert torch.isnan(q[0, :, :2]).all() and torch.isfinite(q[0, :, 2:]).all()
    # the cos / sin caches hold 9 rows: positions 14, 15 are past them, 16, 17 past the table
    assert torch.isnan(q[1]).all()
    own = set(c["table"][1].tolist())
    for p in own:
        assert torch.equal(vc[p].cpu(), c["vc"][p])
    c = _case(T=4, starts=(0, 5), seed=8)
    c["table"][0, 0] = c["kc"].size(0)
    c["table"][1, 0] = -1
    q, kc, vc = _run(c)
    assert torch.isnan(q.float()).all()
    assert torch.equal(kc.cpu(), c["kc"]) and torch.equal(vc.cpu(), c["vc"])
    assert torch.isfinite(good[0].float()).all()


def test_token_major_cache_and_slices():
    c = _case(T=6, starts=(3, 20), seed=9)
    want = _run(c)
    d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    P, U, ps, hd = c["kc"].shape
    pool = torch.zeros(P, ps, U + c["vc"].size(1), hd, dtype=BF16, device="cuda")
    kc, vc = pool[:, :, :U].transpose(1, 2), pool[:, :, U:].transpose(1, 2)
    kc.copy_(d["kc"])
    vc.copy_(d["vc"])
    q = kernel.paged_append_(d["k"], d["v"], kc, vc, d["table"], d["positions"], q=d["q"], cos=d["cos"][None, None],
                             sin=d["sin"][None, None], q_weight=d["qw"], k_weight=d["kw"], eps=1e-5)
    assert torch.equal(q, want[0]) and torch.equal(kc, want[1]) and torch.equal(vc, want[2])


def test_zero_tokens():
    c = _case(seed=10)
    d = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    q = kernel.paged_append_(d["k"][:, :, :0], d["v"][:, :, :0], d["kc"], d["vc"], d["table"], d["positions"],
                             q=d["q"][:, :, :0], cos=d["cos"], sin=d["sin"])
    assert q.shape == (2, 4, 0, 64) and torch.equal(d["kc"].cpu(), c["kc"])
