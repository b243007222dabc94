"""Every form of the single-token attention kernel against float64: whole
sequences on four and on eight waves, and key ranges with their join, at each
head dim and type, without groups and with KV groups of 1 to 17 columns (the
largest requests for LDS among them)."""
import pytest
import torch

import kernel
from decode_cases import paged_case, paged_reference, paged_tolerance, run_paged
from kernel import _ext
from test_decode_refusals import T as _desc, _attn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HDS, DTYPES = [32, 64, 96, 128, 256], [BF16, FP16, FP32]


def _widen(c, positions):
    """The same sequences behind a table of so many positions."""
    n = -(-positions // c["page"])
    if n > c["table"].size(1):
        wide = torch.full((c["table"].size(0), n), -1, dtype=torch.int32)
        wide[:, :c["table"].size(1)] = c["table"]
        c["table"] = wide
    return c


def _is_cut(c):
    """Whether the call deals its keys out in ranges (needs a workspace)."""
    code = _ext._DTYPE_CODE
    kw = {n: _desc(tuple(c[t].shape), code[c[t].dtype]) for n, t in
          (("q", "q"), ("k_cache", "kc"), ("v_cache", "vc"), ("page_table", "table"), ("lengths", "lengths"), ("alpha", "alpha"),
           ("rho", "rho"), ("z", "z"), ("patt", "patt")) if c[t] is not None and c[t].numel()}
    B, H = c["lengths"].numel(), c["frozen"].numel()
    a, keep = _attn(H=H, out=_desc((B, H, 1, c["hd"]), code[c["vc"].dtype]), frozen=c["frozen"].tolist(),
                    hidx=c["hidx"].tolist(), pidx=c["pidx"].tolist(),
                    kvidx=None if c["kvidx"] is None else c["kvidx"].tolist(), **kw)
    n = _ext.lib().saf_paged_attn_workspace_bytes(a)
    assert n >= 0 and keep is not None
    return n > 0


def _check(c, cut):
    assert _is_cut(c) == cut
    lse = torch.zeros(c["lengths"].numel(), c["frozen"].numel(), 1, device="cuda")
    out = run_paged(kernel, c, lse=lse).double().cpu()[:, :, 0]
    ref, mag, want = paged_reference(c)
    err, tol = (out - ref).abs(), paged_tolerance(c, ref, mag)
    assert not torch.isnan(out).any()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the bound"
    live = (c["frozen"] == 0) & (c["lengths"][:, None] > 0)
    # base-2 scores of size < 32: a few steps of fp32 there
    assert bool(((lse.double().cpu()[:, :, 0] - want).abs()[live] <= 2.0 ** -15).all())


def _states(H, kinds):
    """Live heads with a frozen one of each kind here and there."""
    s = [0] * H
    for i, k in enumerate(kinds):
        s[(3 * i + 1) % H] = k
    return s


# the columns of one KV head: none shared, 1, 7, 16 and 17 (two units)
GROUPS = [(4, 0), (2, 2), (7, 1), (32, 2), (17, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("H,HKV", GROUPS)
def test_whole_on_four_waves(H, HKV, hd, dtype):
    kinds = (2, 1) if H > 2 else ()
    _check(paged_case([1, 33, 0, 150], H=H, HKV=HKV, hd=hd, dtype=dtype, states=_states(H, kinds), seed=hd + H), cut=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("H,HKV", GROUPS)
def test_ranges_and_join(H, HKV, hd, dtype):
    """Also sequences of less than a range, and an empty one."""
    kinds = (2,) if H > 2 else ()
    c = paged_case([2600, 1, 0, 129, 700], H=H, HKV=HKV, hd=hd, dtype=dtype, page=64, states=_states(H, kinds), seed=hd + H)
    es = 4 if dtype == FP32 else 2
    _check(_widen(c, max(2600, (512 << 10) // (2 * hd * es))), cut=True)


@pytest.mark.parametrize("hd,dtype", [(32, BF16), (32, FP16), (32, FP32), (64, BF16), (64, FP16), (64, FP32), (96, BF16), (96, FP16),
                                      (128, BF16), (128, FP16)])
@pytest.mark.parametrize("H,HKV", [(4, 0), (32, 2), (34, 2)])
def test_whole_on_eight_waves(H, HKV, hd, dtype):
    """Tables of 2048 positions and more, of more sequences than are cut."""
    es, simd = (4, {32: 4, 64: 2}) if dtype == FP32 else (2, {32: 5, 64: 3, 96: 2, 128: 2})
    units = 4 if HKV == 0 or H == 34 else 2
    B = 256 * simd[hd] // units // 2 + 1
    lens = [(37 * i) % 60 + 1 for i in range(B)]
    lens[1], lens[B // 2], lens[-1] = 2048, 300, 1100
    _check(paged_case(lens, H=H, HKV=HKV, hd=hd, dtype=dtype, page=64, states=_states(H, (2,)), seed=hd), cut=False)


@pytest.mark.parametrize("hd,dtype", [(128, BF16), (256, FP16), (256, FP32)])
def test_frozen_groups_of_sixteen(hd, dtype):
    """Sixteen frozen columns, whose weights and partial sums share the LDS."""
    c = paged_case([900, 70], H=16, HKV=1, hd=hd, dtype=dtype, page=64, states=[2] * 15 + [1], seed=hd)
    _check(c, cut=False if c["table"].size(1) * 64 * hd * 2 * (4 if dtype == FP32 else 2) < 512 << 10 else True)
    c = paged_case([900, 70], H=16, HKV=1, hd=hd, dtype=dtype, page=64, states=[0, 1] + [2] * 14, seed=hd)
    _check(_widen(c, 8192), cut=True)


@pytest.mark.parametrize("B", [65, 130])
def test_ranges_of_many_sequences(B):
    """More sequences than a wave has lanes."""
    lens = [(53 * i) % 400 for i in range(B)]
    lens[0], lens[B - 1] = 3000, 1500
    _check(paged_case(lens, H=7, HKV=1, hd=64, page=64, states=_states(7, (2,)), seed=B), cut=True)
