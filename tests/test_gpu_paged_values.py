"""Single-token attention over values that are not finite, against float64:
infinities reach their own element of the result and no other."""
import pytest
import torch

import kernel
from decode_cases import paged_case, paged_reference, paged_tolerance, run_paged

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")


def _put(c, b, pos, head, d, value):
    """Value d of head (all heads: None) of sequence b's token at pos."""
    pg, sl = int(c["table"][b, pos // c["page"]]), pos % c["page"]
    c["vc"][pg, slice(None) if head is None else head, sl, d] = value


def _check(c):
    out = run_paged(kernel, c).double().cpu()[:, :, 0]
    ref, mag, _ = paged_reference(c)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(out[~fin].nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0), ref[~fin].nan_to_num(nan=0.0, posinf=1.0, neginf=-1.0))
    finite = dict(c, vc=torch.where(torch.isfinite(c["vc"]), c["vc"], torch.zeros((), dtype=c["vc"].dtype)))
    tol = paged_tolerance(finite, ref, mag)
    assert bool(((out - ref).abs() <= tol)[fin].all())
    return ref


# one key range of one to seven steps, and (the last two) several ranges
LENS = [[1, 17], [33, 48], [200, 5], [6000, 3], [2500, 2100]]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("HKV", [0, 2])
@pytest.mark.parametrize("lens", LENS)
def test_infinite_values(lens, HKV, dtype):
    """Both signs, the newest token's among them, one element each."""
    c = paged_case(lens, H=4, HKV=HKV, page=64 if lens[0] > 1000 else 16, dtype=dtype, states=[0, 2, 1 if lens[0] < 1000 else 0, 0],
                   seed=lens[0])
    n = lens[0]
    _put(c, 0, n - 1, None, 3, INF)
    _put(c, 0, 0, 1, 9, -INF)
    _put(c, 0, n // 2, 0, 40, -INF)
    _put(c, 1, lens[1] - 1, 0, 63, INF)
    ref = _check(c)
    assert int(torch.isinf(ref).sum()) >= 6


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [70, 5000])
def test_both_signs_and_nan(n, dtype):
    c = paged_case([n, 9], H=3, page=64, dtype=dtype, states=[0, 2, 0], seed=n)
    _put(c, 0, 1, None, 5, INF)
    _put(c, 0, n - 2, None, 5, -INF)
    _put(c, 0, n - 3, 2, 6, float("nan"))
    _put(c, 0, 7, None, 30, INF)
    _put(c, 0, n - 1, None, 30, INF)
    ref = _check(c)
    assert torch.isnan(ref[0, :, 5]).all() and torch.isnan(ref[0, 2, 6]) and torch.isinf(ref[0, :, 30]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_weights_of_zero_and_below(dtype):
    """A dense pattern's weight 0 makes an infinite value NaN, a negative
    weight turns its sign."""
    c = paged_case([40, 20], H=2, dtype=dtype, states=[1, 0], seed=3)
    c["patt"][0, 39, 4], c["patt"][0, 39, 5] = 0.0, -0.25
    _put(c, 0, 4, 0, 10, INF)
    _put(c, 0, 5, 0, 11, INF)
    ref = _check(c)
    assert torch.isnan(ref[0, 0, 10]) and float(ref[0, 0, 11]) == -INF


def test_infinite_values_do_not_hide_other_faults():
    """A bad page, a pattern that is too short, a NaN weight: NaN as before."""
    c = paged_case([60, 61, 62, 50], states=[0, 2, 0, 1], page=16, seed=12, S=61)
    for b, n in enumerate((60, 61, 62, 50)):
        _put(c, b, n - 1, None, 0, INF)
    c["table"][0, 1] = c["kc"].size(0)
    c["lengths"][3] = 16 * c["table"].size(1) + 1
    c["alpha"][1, 7] = float("nan")
    out = run_paged(kernel, c).float().cpu()[:, :, 0]
    assert torch.isnan(out[0]).all() and torch.isnan(out[3]).all()
    assert torch.isnan(out[1, 1]).all() and torch.isnan(out[2, [1, 3]]).all()
    assert torch.isinf(out[1, [0, 2], 0]).all() and torch.isinf(out[2, [0, 2], 0]).all()
    assert torch.isfinite(out[1, [0, 2], 1:]).all()
