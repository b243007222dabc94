"""gelu_packed and mlp_packed where no gradient is recorded: the same results, and no
8 bits that nothing would read."""
import pytest
import torch

import kernel
from kernel import _ext
from test_train_ops_refusals import _BF16, _I8, _NONE, _U8, _refused, _t

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def test_entry_point():
    """q and exp are absent together (no rows: nothing is launched)."""
    L = _ext.lib()
    x, q, e = _t((0, 40), _BF16), _t((0, 40), _I8), _t((0, 2), _U8)
    assert L.saf_gelu_pack_fwd(x, x, _NONE, _NONE, None) == _ext.SAF_OK
    assert L.saf_gelu_pack_fwd(x, x, None, None, None) == _ext.SAF_OK
    _refused(L.saf_gelu_pack_fwd(x, x, q, _NONE, None), _ext.SAF_EINVAL, "exp is required")
    _refused(L.saf_gelu_pack_fwd(x, x, _NONE, e, None), _ext.SAF_EINVAL, "q is required")
    _refused(L.saf_act_pack(x, _NONE, _NONE, None), _ext.SAF_EINVAL, "q is required")
    _refused(L.saf_gelu_pack_bwd(_NONE, _NONE, x, x, _NONE, None), _ext.SAF_EINVAL, "q is required")


def _peak(f):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    f()
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("R,C", [(1, 1), (3, 33), (130, 2048), (257, 2001)])
def test_same_results(dtype, R, C):
    x = torch.randn(R, C, device="cuda", generator=torch.Generator("cuda").manual_seed(C)).mul_(3).to(dtype)
    x.view(-1)[::97] = float("inf")
    x.view(-1)[5::101] = float("nan")
    want = kernel.gelu_packed(x.clone().requires_grad_()).detach()
    wide = torch.zeros(R, C + 3, device="cuda", dtype=dtype)[:, 1:C + 1]
    wide.copy_(x)
    got = [kernel.gelu_packed(x), kernel.gelu_packed(wide)]
    with torch.no_grad():
        got.append(kernel.gelu_packed(x.clone().requires_grad_()))
    for y in got:
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.mark.gpu
def test_nothing_is_packed():
    n = 1 << 22
    x = torch.randn(1 << 12, 1 << 10, device="cuda", dtype=BF16)
    assert _peak(lambda: kernel.gelu_packed(x)) <= 2 * n + 4096
    w1, w2 = torch.randn(4096, 1024, device="cuda", dtype=BF16), torch.randn(1024, 4096, device="cuda", dtype=BF16)
    kernel.mlp_packed(x, w1, w2)                             # workspaces of the products
    hidden = 2 * (2 * 4 * n)                                 # the GELU's input and output
    assert _peak(lambda: kernel.mlp_packed(x, w1, w2)) <= hidden + 4096
    leaves = [t.clone().requires_grad_() for t in (w1, w2)]
    want = kernel.mlp_packed(x, *leaves).detach()
    with torch.no_grad():
        assert _peak(lambda: kernel.mlp_packed(x, *leaves)) <= hidden + 4096
        assert torch.equal(kernel.mlp_packed(x, *leaves), want)
