"""What the operators around the products of a training step refuse, on the CPU:
before any device is looked at, or with addresses that no kernel gets to see."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

import kernel
from kernel import _ext

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def test_cpu_tensors_are_refused():
    w, x = torch.zeros(4, 8), torch.zeros(2, 8)
    for call in (lambda: kernel.embed_tokens(torch.zeros(2, dtype=torch.long), w),
                 lambda: kernel.add_layernorm(x, None, w[0]), lambda: kernel.gelu_packed(x),
                 lambda: kernel.pack_activation(x), lambda: kernel.mlp_packed(x, torch.zeros(32, 8), torch.zeros(8, 32)),
                 lambda: kernel.unpack_activation(kernel.PackedActivation(x.to(torch.int8), x.to(torch.uint8), F32))):
        with pytest.raises(RuntimeError, match="HIP devices only"):
            call()


def test_tangents_are_refused():
    x, w, t = torch.zeros(2, 8), torch.zeros(8), torch.zeros(2, dtype=torch.long)
    with fwd.dual_level():
        dual, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, w)
        for call in (lambda: kernel.embed_tokens(t, dual), lambda: kernel.add_layernorm(dual, None, w),
                     lambda: kernel.add_layernorm(x, dual, w), lambda: kernel.add_layernorm(x, None, dw),
                     lambda: kernel.add_layernorm(x, None, w, dw), lambda: kernel.gelu_packed(dual),
                     lambda: kernel.pack_activation(dual),
                     lambda: kernel.mlp_packed(dual, torch.zeros(32, 8), torch.zeros(8, 32))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="no forward-mode"):
                    call()


def test_dtypes_that_no_operator_has():
    w = torch.zeros(4, 8)
    for dt in (torch.float64, torch.int32, torch.int64):
        with pytest.raises(NotImplementedError, match="unsupported dtype"):
            kernel.embed_tokens(torch.zeros(2, dtype=torch.long), w, dtype=dt)
        with pytest.raises(NotImplementedError, match="unsupported dtype"):
            kernel.add_layernorm(w, None, w[0], dtype=dt)


def test_mlp_shapes():
    x = torch.zeros(2, 8)
    for fc, proj in (((32, 9), (8, 32)), ((32, 8), (8, 31)), ((32, 8, 1), (8, 32))):
        with pytest.raises(ValueError, match="mlp_packed takes x"):
            kernel.mlp_packed(x, torch.zeros(fc), torch.zeros(proj))
    with pytest.raises(ValueError, match="one dtype"):
        kernel.mlp_packed(x, torch.zeros(32, 8, dtype=BF16), torch.zeros(8, 32))


def _t(shape, code, stride=None, ptr=0x100000):
    d = _ext.SafTensor()
    d.data, d.dtype, d.ndim = ptr, code, len(shape)
    st = [1] * len(shape)
    for i in range(len(shape) - 2, -1, -1):
        st[i] = st[i + 1] * shape[i + 1]
    for i, n in enumerate(shape):
        d.size[i] = n
        d.stride[i] = (stride or st)[i]
    return d


_NONE = _ext.SafTensor()
_F32, _F16, _BF16, _I32, _I64, _I8, _U8 = (getattr(_ext, "SAF_" + n) for n in ("F32", "F16", "BF16", "I32", "I64", "I8", "U8"))


def _refused(rc, code, text):
    assert rc == code, (rc, _ext.lib().saf_last_error())
    assert text in _ext.lib().saf_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(tokens=_t((3,), _F32)), _ext.SAF_EINVAL, "tokens must be int32 or int64"),
    (dict(tokens=_t((3, 1), _I64)), _ext.SAF_EINVAL, "tokens must be int32 or int64"),
    (dict(weight=_t((9, 16), _I32)), _ext.SAF_EUNSUPPORTED, "unsupported dtype int32"),
    (dict(weight=_t((0, 16), _BF16)), _ext.SAF_EINVAL, "rows and channels"),
    (dict(weight=_t((9, 16), _BF16, (16, 2))), _ext.SAF_EALIGN, "unit column stride"),
    (dict(out=_t((3, 15), _BF16)), _ext.SAF_EINVAL, "out must be (3, 16)"),
    (dict(out=_t((3, 16), _BF16, (32, 1))), _ext.SAF_EALIGN, "out must be contiguous"),
    (dict(out=_t((3, 16), _F16)), _ext.SAF_EUNSUPPORTED, "bf16 beside fp16"),
    (dict(weight=_t((9, 16), _BF16, ptr=0x100001)), _ext.SAF_EALIGN, "not aligned to its elements"),
    (dict(tokens=_t((1 << 31,), _I32), out=_t((1 << 31, 16), _BF16)), _ext.SAF_EUNSUPPORTED, "2^31 groups"),
])
def test_embed_arguments(change, code, text):
    a = dict(dict(tokens=_t((3,), _I64), weight=_t((9, 16), _BF16), out=_t((3, 16), _BF16)), **change)
    _refused(_ext.lib().saf_embed_fwd(a["tokens"], a["weight"], 1.0, -100, a["out"], None), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(dout=_t((301, 16), _BF16)), _ext.SAF_EINVAL, "dout must be (300, 16)"),
    (dict(dout=_t((300, 16), _F16)), _ext.SAF_EUNSUPPORTED, "bf16 beside fp16"),
    (dict(dweight=_t((9, 16), _BF16, (32, 1))), _ext.SAF_EALIGN, "dweight must be contiguous"),
    (dict(dweight=_t((9, 16), _BF16, ptr=0x100008)), _ext.SAF_EALIGN, "dweight must be 16-byte aligned"),
    (dict(ws=None), _ext.SAF_EWORKSPACE, "workspace"),
    (dict(ws=0x100080), _ext.SAF_EALIGN, "256-byte aligned"),
    (dict(short=1), _ext.SAF_EWORKSPACE, "workspace"),
])
def test_embed_bwd_arguments(change, code, text):
    L = _ext.lib()
    a = dict(dict(dout=_t((300, 16), _BF16), dweight=_t((9, 16), _BF16), ws=0x100000, short=0), **change)
    n = L.saf_embed_bwd_workspace_bytes(300, 9, 16) - a["short"]
    _refused(L.saf_embed_bwd(_t((300,), _I64), a["dout"], 1.0, -100, a["dweight"], a["ws"], n, None), code, text)


def test_embed_bwd_sizes():
    """More threads than a launch has are refused, not cut short."""
    L, n, C = _ext.lib(), 1 << 28, 8192
    _refused(L.saf_embed_bwd(_t((n,), _I64), _t((n, C), _BF16), 1.0, -100, _t((9, C), _BF16), 0x100000, 1 << 60, None),
             _ext.SAF_EUNSUPPORTED, "too many tokens")
    _refused(L.saf_embed_bwd(_t((n + 1,), _I64), _t((n + 1, 8), _BF16), 1.0, -100, _t((9, 8), _BF16), 0x100000, 1 << 60, None),
             _ext.SAF_EUNSUPPORTED, "at most 2^28")


def test_embed_workspace():
    f = _ext.lib().saf_embed_bwd_workspace_bytes
    assert f(0, 9, 16) == 0 and f(65, 9, 16) > 8 * 65
    assert f(3, 9, 16) == f(64, 9, 16) == 0          # nothing is sorted
    assert f(-1, 9, 16) == f(3, 0, 16) == f(3, 9, 0) == f((1 << 28) + 1, 9, 16) == f(3, 1 << 31, 16) == -1
    # a second buffer and digit counts only with several tiles (and passes)
    assert f(8193, 600, 8) - f(8193, 500, 8) == (8 * 8193 + 255) // 256 * 256
    assert f(8192, 600, 8) == f(8192, 500, 8)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=_t((3, 16), _I32)), _ext.SAF_EUNSUPPORTED, "unsupported dtype int32"),
    (dict(x=_t((3, 16385), _BF16)), _ext.SAF_EUNSUPPORTED, "C = 16385"),
    (dict(x=_t((3, 0), _BF16)), _ext.SAF_EUNSUPPORTED, "C = 0"),
    (dict(x=_t((1 << 29, 16), _BF16)), _ext.SAF_EUNSUPPORTED, "too many rows"),
    (dict(x=_t((1 << 22, 16384), _BF16)), _ext.SAF_EUNSUPPORTED, "too many rows"),
    (dict(y=_t((3, 16), _F32)), _ext.SAF_EUNSUPPORTED, "bfloat16 x with float32 y"),
    (dict(x=_t((3, 16), _F16)), _ext.SAF_EUNSUPPORTED, "float16 x with bfloat16 y"),
    (dict(delta=_t((3, 16), _F32)), _ext.SAF_EINVAL, "r must have x's dtype and delta y's"),
    (dict(delta=_t((2, 16), _BF16)), _ext.SAF_EINVAL, "delta must be (3, 16)"),
    (dict(r=_NONE), _ext.SAF_EINVAL, "delta and r go together"),
    (dict(weight=_t((15,), _F32)), _ext.SAF_EINVAL, "weight must be a contiguous floating (16,) vector"),
    (dict(bias=_t((16,), _BF16)), _ext.SAF_EINVAL, "of the weight's dtype"),
    (dict(stats=_t((3, 2), _BF16)), _ext.SAF_EINVAL, "stats must be fp32"),
    (dict(eps=-1.0), _ext.SAF_EINVAL, "eps"),
    (dict(eps=float("nan")), _ext.SAF_EINVAL, "eps"),
])
def test_layernorm_arguments(change, code, text):
    a = dict(dict(x=_t((3, 16), _BF16), delta=_t((3, 16), _BF16), weight=_t((16,), _F32), bias=_t((16,), _F32), eps=1e-5,
                  r=_t((3, 16), _BF16), y=_t((3, 16), _BF16), stats=_t((3, 2), _F32)), **change)
    _refused(_ext.lib().saf_layernorm_fwd(a["x"], a["delta"], a["weight"], a["bias"], a["eps"], a["r"], a["y"], a["stats"], None),
             code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(dy=_t((300, 16), _F32)), _ext.SAF_EUNSUPPORTED, "bfloat16 r with float32 dy"),
    (dict(stats=_NONE), _ext.SAF_EINVAL, "stats is required"),
    (dict(dr=_t((300, 16), _F32)), _ext.SAF_EINVAL, "dr and dx must have r's dtype"),
    (dict(dx=_t((300, 16), _BF16, (20, 1))), _ext.SAF_EALIGN, "dx must be contiguous"),
    (dict(ddelta=_t((300, 16), _F32)), _ext.SAF_EINVAL, "ddelta must have dy's dtype"),
    (dict(dw=_t((16,), _BF16)), _ext.SAF_EINVAL, "of the weight's dtype"),
    (dict(ws=None), _ext.SAF_EWORKSPACE, "workspace"),
    (dict(ws=0x100010), _ext.SAF_EALIGN, "256-byte aligned"),
])
def test_layernorm_bwd_arguments(change, code, text):
    a = dict(dict(dy=_t((300, 16), _BF16), stats=_t((300, 2), _F32), dr=_NONE, dx=_t((300, 16), _BF16), ddelta=_NONE,
                  dw=_t((16,), _F32), ws=0x100000), **change)
    L = _ext.lib()
    n = L.saf_layernorm_bwd_workspace_bytes(300, 16)
    assert n > 0
    _refused(L.saf_layernorm_bwd(_t((300, 16), _BF16), a["stats"], _t((16,), _F32), a["dy"], a["dr"], a["dx"], a["ddelta"],
                                 a["dw"], _NONE, a["ws"], n, None), code, text)


def test_layernorm_workspace():
    f = _ext.lib().saf_layernorm_bwd_workspace_bytes
    assert f(0, 16) == 0
    assert f(-1, 16) == f(3, 0) == f(3, 16385) == -1
    assert f(1, 16) == f(128, 16) == 0 and f(129, 16) == 5 * 2 * 16 * 4    # rounds of 32 rows, four by one workgroup


@pytest.mark.parametrize("change,code,text", [
    (dict(x=_t((3, 40), _I8)), _ext.SAF_EUNSUPPORTED, "unsupported dtype int8"),
    (dict(x=_t((40,), _BF16)), _ext.SAF_EINVAL, "2-D"),
    (dict(q=_t((3, 40), _U8)), _ext.SAF_EINVAL, "q must be int8 and exp uint8"),
    (dict(q=_t((3, 39), _I8)), _ext.SAF_EINVAL, "q must be (3, 40)"),
    (dict(exp=_t((3, 1), _U8)), _ext.SAF_EINVAL, "exp must be (3, 2)"),
    (dict(q=_t((3, 40), _I8, (64, 1))), _ext.SAF_EALIGN, "q must be contiguous"),
    (dict(y=_t((3, 40), _F32)), _ext.SAF_EINVAL, "y must have x's dtype"),
])
def test_packed_arguments(change, code, text):
    L = _ext.lib()
    a = dict(dict(x=_t((3, 40), _BF16), q=_t((3, 40), _I8), exp=_t((3, 2), _U8), y=_t((3, 40), _BF16)), **change)
    _refused(L.saf_gelu_pack_fwd(a["x"], a["y"], a["q"], a["exp"], None), code, text)
    _refused(L.saf_act_unpack(_t((3, 40), _I8), _t((3, 2), _U8), _t((3, 40), _BF16, (39, 1)), None), _ext.SAF_EINVAL, "overlap")
    if "y" not in change:
        _refused(L.saf_act_pack(a["x"], a["q"], a["exp"], None), code, text)
        _refused(L.saf_act_unpack(a["q"], a["exp"], a["x"], None), code, text.replace("x", "out") if "2-D" in text else text)
