"""Forward-mode tangents are refused, not dropped, by the decoding operators
(CPU: before any device is looked at; the same checks run on the device)."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

import kernel
from kernel import _ext, paged

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_token_logprobs(device, grad):
    x, t = torch.randn(3, 50, device=device, requires_grad=grad), torch.zeros(3, dtype=torch.long, device=device)
    with fwd.dual_level():
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError, match="no forward-mode"):
                _ext.bind().token_logprobs(fwd.make_dual(x, torch.ones_like(x)), t, 0, False, 1.0, -100)
        # unpacked, or where forward mode is off: nothing to refuse
        if device == "cuda":
            dual = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="no forward-mode"):
                kernel.token_logprobs(dual.view(1, 3, 50), t.view(1, 3))
            assert kernel.token_logprobs(fwd.unpack_dual(dual).primal, t).logp.shape == (3,)
            with torch.inference_mode():
                assert kernel.token_logprobs(x, t).logp.shape == (3,)


@pytest.mark.parametrize("device", DEVICES)
def test_descriptors(device):
    args = _ext.SafPagedAttnArgs()
    x = torch.zeros(1, 2, 1, 64, device=device)
    at = paged._ATTN_AT[:1]
    with fwd.dual_level(), torch.no_grad():
        for refuse in (True, False):
            with pytest.raises(NotImplementedError, match="attention has no forward-mode"):
                _ext.bind().fill("attention", ctypes.addressof(args), at, 0, 0, refuse, fwd.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
def test_paged_operators():
    kc = torch.zeros(3, 2, 16, 64, device="cuda")
    table, one = torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    x, frozen = torch.zeros(1, 2, 1, 64, device="cuda"), torch.zeros(2, dtype=torch.int32)
    w = torch.ones(64, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="paged_mixed_attn has no forward-mode"):
            kernel.paged_mixed_attn(dual, kc, kc, table, one, None, frozen)
        for kw in (dict(k=dual), dict(v=dual), dict(q=dual), dict(q_weight=fwd.make_dual(w, w), k_weight=w)):
            call = dict(dict(k=x, v=x, q=x), **kw)
            with pytest.raises(NotImplementedError, match="paged_append_ has no forward-mode"):
                kernel.paged_append_(call.pop("k"), call.pop("v"), kc, kc.clone(), table, one, **call)
