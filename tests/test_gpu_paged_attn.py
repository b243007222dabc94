"""Single-token attention over a paged cache against float64, at the sizes,
layouts and lengths where it can go wrong."""
import pytest
import torch

import kernel
from decode_cases import paged_case, paged_reference, paged_tolerance, run_paged

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _check(c, sm_scale=None, **kw):
    out = run_paged(kernel, c, sm_scale=sm_scale, **kw).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c, sm_scale)
    err, tol = (out - ref).abs(), paged_tolerance(c, ref, mag)
    assert not torch.isnan(out).any()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the bound"
    return out


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("lens", [[1], [2, 15, 16, 17], [31, 32, 33, 64, 65], [127, 128, 129, 300]])
def test_lengths_and_head_dims(lens, hd, dtype):
    _check(paged_case(lens, H=4, hd=hd, dtype=dtype, states=[0, 2, 1, 0], seed=hd))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("H,HKV", [(14, 2), (8, 8), (32, 8), (7, 1), (16, 1), (17, 1), (40, 2), (128, 4)])
def test_groups(H, HKV, dtype):
    """Group sizes below, at and above one unit's 16 columns."""
    _check(paged_case([100, 37], H=H, HKV=HKV, dtype=dtype, seed=H))


@pytest.mark.parametrize("states", [[0, 0, 2, 1, 0, 2, 0], [2] * 7, [1, 1, 1, 1, 1, 1, 1], [0] * 6 + [1], [2, 1, 2, 1, 2, 1, 0]])
@pytest.mark.parametrize("HKV", [0, 1])
def test_head_states(states, HKV):
    _check(paged_case([1, 33, 200], H=7, HKV=HKV, states=states, seed=3))


@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_page_sizes(page):
    _check(paged_case([1, page - 1, page, page + 1, 3 * page + 5], page=page, states=[0, 2, 0, 0], seed=page))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("HKV", [0, 2])
def test_long_and_split(dtype, HKV):
    """Few sequences of very different lengths: key ranges joined."""
    _check(paged_case([9000, 1, 257, 4096], H=4, HKV=HKV, hd=64, page=64, dtype=dtype, states=[0, 2, 0, 0], seed=9))


def test_many_sequences():
    lens = [(37 * i) % 190 + 1 for i in range(300)]
    _check(paged_case(lens, H=4, HKV=2, hd=32, states=[0, 0, 2, 0], seed=1))


def test_empty_sequences():
    c = paged_case([0, 5, 0, 700], states=[0, 1, 2, 0], seed=4)
    lse = torch.full((4, 4, 1), 7.0, device="cuda")
    out = run_paged(kernel, c, lse=lse)
    ref, mag, rl = paged_reference(c)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    got = out.double().cpu()[:, :, 0]
    assert bool(((got - ref).abs() <= paged_tolerance(c, ref, mag)).all())
    live = c["frozen"] == 0
    l = lse.cpu().double()[:, :, 0]
    assert (l[0, live] == -float("inf")).all()
    fin = torch.isfinite(rl) & live
    # base-2 scores of size < 16: a few steps of fp32 at 16
    assert bool(((l - rl).abs()[fin] <= 2.0 ** -16).all())
    assert (l[:, ~live] == 7.0).all()       # frozen heads' entries are left alone


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (FP16, 16), (FP32, 17)])
@pytest.mark.parametrize("lens", [[70, 200], [5000, 1]])
def test_lse(lens, dtype, bits):
    """Base-2 log-sum-exp of the live heads (values below 16: a few fp32 steps),
    whole and joined."""
    c = paged_case(lens, H=4, HKV=2, dtype=dtype, page=64, states=[0, 2, 0, 0], seed=21)
    lse = torch.zeros(2, 4, 1, device="cuda")
    run_paged(kernel, c, lse=lse)
    _, _, want = paged_reference(c)
    live = c["frozen"] == 0
    assert bool(((lse.cpu().double()[:, :, 0] - want).abs()[:, live] <= 2.0 ** -bits).all())


@pytest.mark.parametrize("lens", [[3000, 40], [40, 41]])
def test_many_frozen_columns(lens):
    """A group whose frozen weights exceed the LDS block: the keys in turns."""
    _check(paged_case(lens, H=16, HKV=1, page=64, states=[0] + [2] * 15, seed=22))
    _check(paged_case(lens, H=16, HKV=1, page=64, states=[2] * 16, dtype=FP16, seed=23))


def test_wide_table_of_short_sequences():
    """A table far wider than the sequences: the ranges follow the lengths."""
    c = paged_case([300, 700], H=2, seed=24)
    wide = torch.full((2, 2000), -1, dtype=torch.int32)
    wide[:, :c["table"].size(1)] = c["table"]
    c["table"] = wide
    _check(c)


def test_large_uncut_batch():
    """More units than resident workgroups, long enough for eight waves."""
    lens = [(331 * i) % 2100 + 1 for i in range(160)]
    _check(paged_case(lens, H=8, HKV=8, hd=32, page=64, states=[0, 2, 0, 0, 0, 1, 0, 0], seed=25))


@pytest.mark.parametrize("patt_dtype", [FP32, BF16, FP16])
def test_pattern_types(patt_dtype):
    _check(paged_case([130, 64, 3], states=[1, 0, 1, 1], patt_dtype=patt_dtype, seed=5))


def test_identity_tables_and_scale():
    c = paged_case([77, 5], H=3, seed=6)
    c["hidx"] = c["pidx"] = None
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    out = kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], sm_scale=-0.3)
    c["hidx"] = torch.arange(3)
    ref, mag, _ = paged_reference(c, -0.3)
    assert bool(((out.double().cpu()[:, :, 0] - ref).abs() <= paged_tolerance(c, ref, mag)).all())


def test_decomposed_without_z():
    c = paged_case([50, 20], states=[0, 2, 2, 0], seed=7)
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    out = kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"],
                                  alpha=m["alpha"], rho=m["rho"])
    ref, mag, _ = paged_reference(c)
    assert bool(((out.double().cpu()[:, :, 0] - ref).abs() <= paged_tolerance(c, ref, mag)).all())


def test_large_pattern_logits():
    """Logits of size 150: the sum's rounding alone (2^-24 150 = 9e-6 of the
    weight) would show in float32; what is left is exp2's argument (2^-24 of
    its size where the weight matters, below 40) and a few roundings."""
    c = paged_case([300, 77], H=3, states=[2, 0, 2], dtype=FP32, seed=26)
    c["alpha"] *= 80
    c["rho"] *= 80
    c["z"] = torch.stack([torch.logsumexp(c["alpha"][:, :n].double() + c["rho"][:, :n].flip(1).double(), 1)
                          for n in range(1, 301)], 1).float()
    out = run_paged(kernel, c).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c)
    assert bool(((out - ref).abs() <= 2.0 ** -17 * mag + 2.0 ** -24 * ref.abs())[:, [0, 2]].all())


def test_window_pattern():
    """rho = -inf past a window: exact zeros for the far keys."""
    c = paged_case([300, 40], states=[2, 0, 2, 0], seed=8)
    c["alpha"].zero_()
    c["rho"].zero_()
    c["rho"][:, 50:] = -float("inf")
    c["z"] = torch.log(torch.clamp(torch.arange(300) + 1.0, max=50.0)).expand(4, 300).contiguous()
    _check(c)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_strides(dtype):
    """Token-major caches, head slices of a larger pool, a wider table."""
    c = paged_case([70, 33], H=4, states=[0, 0, 2, 0], dtype=dtype, seed=10)
    want = run_paged(kernel, c)
    P, U, ps, hd = c["kc"].shape
    d = dict(c)
    d["kc"] = torch.full((P, ps, U + 2, hd), float("nan"), dtype=dtype)[:, :, 1:U + 1].transpose(1, 2).copy_(c["kc"])
    P, Hv, ps, hd = c["vc"].shape
    d["vc"] = torch.full((2 * P, ps, Hv, 2 * hd), float("nan"), dtype=dtype)[::2, :, :, hd:].transpose(1, 2).copy_(c["vc"])
    d["table"] = torch.full((4, 20), -7, dtype=torch.int32)[::2]
    d["table"][:, :c["table"].size(1)] = c["table"]
    q = torch.full((2, 6, 3, hd), float("nan"), dtype=dtype)[:, 1:4, 1:2]
    d["q"] = q.copy_(c["q"])
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in d.items()}
    # .cuda() keeps dense strides only: lay the views out again on the device
    m["kc"] = torch.full((P, ps, U + 2, hd), float("nan"), dtype=dtype, device="cuda")[:, :, 1:U + 1].transpose(1, 2)
    m["kc"].copy_(c["kc"])
    m["vc"] = torch.full((2 * P, ps, Hv, 2 * hd), float("nan"), dtype=dtype, device="cuda")[::2, :, :, hd:].transpose(1, 2)
    m["vc"].copy_(c["vc"])
    wide = torch.full((4, 20), -7, dtype=torch.int32, device="cuda")
    m["table"] = wide[::2]
    m["table"].copy_(d["table"])
    m["q"] = torch.full((2, 6, 3, hd), float("nan"), dtype=dtype, device="cuda")[:, 1:4, 1:2]
    m["q"].copy_(c["q"])
    got = kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"],
                                  alpha=m["alpha"], rho=m["rho"], z=m["z"])
    ref, mag, _ = paged_reference(c)
    tol = paged_tolerance(c, ref, mag)
    assert bool(((got.double().cpu()[:, :, 0] - ref).abs() <= tol).all())
    assert bool(((want.double().cpu()[:, :, 0] - ref).abs() <= tol).all())


def test_misaligned_query_rows():
    c = paged_case([40], H=2, hd=64, seed=11)
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    buf = torch.zeros(2 * 64 + 1, dtype=BF16, device="cuda")
    q = buf[1:].view(1, 2, 1, 64)
    q.copy_(m["q"])
    out = kernel.paged_mixed_attn(q, m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"])
    ref, mag, _ = paged_reference(c)
    assert bool(((out.double().cpu()[:, :, 0] - ref).abs() <= paged_tolerance(c, ref, mag)).all())


@pytest.mark.parametrize("cap_pages", [None, 40])
def test_bad_pages_and_lengths_give_nan(cap_pages):
    """Ids outside the cache and lengths past the table or a pattern poison
    their own rows and no other (few pages: one key range; many: several)."""
    c = paged_case([60, 61, 62, 50], states=[0, 2, 0, 1], page=16, seed=12, S=61)
    if cap_pages:
        wide = torch.full((4, cap_pages), -1, dtype=torch.int32)
        wide[:, :c["table"].size(1)] = c["table"]
        c["table"] = wide
    good = run_paged(kernel, c).float().cpu()
    assert torch.isfinite(good[0]).all() and torch.isfinite(good[3]).all()
    # length 62 on patterns of 61 rows: the frozen heads only
    assert torch.isnan(good[2][[1, 3]]).all() and torch.isfinite(good[2][[0, 2]]).all()
    c["table"][0, 1] = c["kc"].size(0)
    c["lengths"][3] = 16 * c["table"].size(1) + 1
    out = run_paged(kernel, c).float().cpu()
    assert torch.isnan(out[0]).all() and torch.isnan(out[3]).all()
    assert torch.equal(out[1], good[1])
    c["table"][0, 1] = -1
    c["lengths"][1] = -5
    out = run_paged(kernel, c).float().cpu()
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()


def test_infinite_scores_and_values():
    """A key of score -inf has weight 0; only a NaN or +inf of a held token
    reaches the result."""
    c = paged_case([40], H=1, seed=13)
    c["q"] = c["q"].abs() + 0.5
    first = int(c["table"][0, 0])
    c["kc"][first, 0, 3] = -float("inf")
    _check_like = run_paged(kernel, c).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c)
    assert bool(((_check_like - ref).abs() <= paged_tolerance(c, ref, mag)).all())
    c["kc"][first, 0, 3] = float("nan")
    assert torch.isnan(run_paged(kernel, c).float()).all()


def test_first_keys_at_minus_infinity():
    """A whole step of -inf scores before the first finite one."""
    c = paged_case([100], H=1, page=16, seed=14)
    c["q"] = c["q"].abs() + 0.5
    for p in range(4):
        c["kc"][int(c["table"][0, p]), 0] = -float("inf")
    out = run_paged(kernel, c).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c)
    assert bool(((out - ref).abs() <= paged_tolerance(c, ref, mag)).all())


def test_large_scores():
    """Peaked softmax: the running maximum moves by hundreds."""
    c = paged_case([500, 90], H=2, seed=15, qscale=30.0)
    out = run_paged(kernel, c).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c)
    # scores up to ~1000: the fp32 sum's rounding moves weights by 1000 66 2^-24
    tol = paged_tolerance(c, ref, mag) + 2 * 1000 * 66 * 2.0 ** -24 * mag
    assert bool(((out - ref).abs() <= tol).all())


def test_same_answer_twice():
    c = paged_case([3000, 17], H=4, HKV=2, states=[0, 2, 0, 0], seed=16)
    assert torch.equal(run_paged(kernel, c), run_paged(kernel, c))


def test_shared_page():
    """A page in two sequences' tables (a common prefix)."""
    c = paged_case([40, 40], H=2, seed=17)
    c["table"][1, :2] = c["table"][0, :2]
    _check(c)


def test_gradients_are_refused():
    c = paged_case([20], H=2, seed=18)
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    q = m["q"].requires_grad_()
    with pytest.raises(NotImplementedError, match="no backward"):
        kernel.paged_mixed_attn(q, m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"])
    with torch.no_grad():
        out = kernel.paged_mixed_attn(q, m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"])
    assert not out.requires_grad
    v = m["vc"].new_zeros(1, 2, 1, 64).requires_grad_()
    with pytest.raises(NotImplementedError, match="no backward"):
        kernel.paged_append_(v, v, m["kc"], m["vc"], m["table"], m["lengths"])


def test_tensors_of_another_device_are_refused():
    c = paged_case([20], H=2, seed=19)
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    for name in ("q", "kc", "table", "lengths"):
        d = dict(m)
        d[name] = c[name]
        with pytest.raises(ValueError, match="is on cpu"):
            kernel.paged_mixed_attn(d["q"], d["kc"], d["vc"], d["table"], d["lengths"], None, d["frozen"], d["hidx"])
    with pytest.raises(ValueError, match="is on cpu"):
        kernel.token_logprobs(torch.zeros(2, 5, device="cuda"), torch.zeros(2, dtype=torch.long))
    # the routing tables may live on the host
    a = kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"])
    b = kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, c["frozen"], c["hidx"])
    assert torch.equal(a, b)
