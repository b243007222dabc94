"""Refusals of the decoding operators, on the CPU: every one is raised by the
argument checks, before any device work is enqueued (the descriptors point
nowhere)."""
import pytest
import torch

import kernel
from kernel import _ext

PTR = 0x100000
F32, F16, BF16, I32, I64 = _ext.SAF_F32, _ext.SAF_F16, _ext.SAF_BF16, _ext.SAF_I32, _ext.SAF_I64


def T(shape, dtype=BF16, stride=None, ptr=PTR):
    d = _ext.SafTensor()
    d.data, d.dtype, d.ndim = ptr, dtype, len(shape)
    st = stride or [0] * len(shape)
    if stride is None:
        n = 1
        for i in reversed(range(len(shape))):
            st[i] = n
            n *= shape[i]
    for i in range(len(shape)):
        d.size[i], d.stride[i] = shape[i], st[i]
    return d


def _attn(**kw):
    a = _ext.SafPagedAttnArgs()
    H = kw.pop("H", 4)
    base = dict(q=T((2, H, 1, 64)), k_cache=T((9, H, 16, 64)), v_cache=T((9, H, 16, 64)), out=T((2, H, 1, 64)),
                page_table=T((2, 5), I32), lengths=T((2,), I32))
    tables = dict(frozen=[0] * H, hidx=None, pidx=None, kvidx=None)
    scale = kw.pop("sm_scale", 0.125)
    for n, v in kw.items():
        (tables if n in tables else base)[n] = v
    for n, t in base.items():
        if t is not None:
            setattr(a, n, t)
    a.n_heads = H
    keep = [_ext.host_i32(tables[n]) for n in ("frozen", "hidx", "pidx", "kvidx")]
    a.frozen, a.hidx, a.pidx, a.kvidx = keep
    a.sm_scale = scale
    return a, keep


ATTN_BAD = [
    (dict(v_cache=None), "v_cache and out are required", "inval"),
    (dict(v_cache=T((9, 4, 16, 64), I32)), "unsupported v_cache dtype", "unsup"),
    (dict(v_cache=T((9, 4, 16, 80)), k_cache=T((9, 4, 16, 80)), q=T((2, 4, 1, 80)), out=T((2, 4, 1, 80))), "head_dim 80", "unsup"),
    (dict(v_cache=T((9, 4, 24, 64))), "page size 24", "unsup"),
    (dict(v_cache=T((9, 4, 8, 64))), "page size 8", "unsup"),
    (dict(v_cache=T((0, 4, 16, 64))), "no pages", "inval"),
    (dict(v_cache=T((9, 4, 16, 64), stride=[4096, 1024, 32, 1])), "slots overlap", "inval"),
    (dict(v_cache=T((9, 4, 16, 64), stride=[4096, 1024, 68, 1])), "not a multiple of 16 bytes", "align"),
    (dict(v_cache=T((9, 4, 16, 64), ptr=PTR + 2)), "not 16-byte aligned", "align"),
    (dict(v_cache=T((9, 4, 16, 64), stride=[1 << 40, 1 << 36, 1 << 27, 1])), "less than 2 GiB", "unsup"),
    (dict(v_cache=T((9, 3, 16, 64))), "one head per output head", "inval"),
    (dict(k_cache=T((9, 3, 16, 64))), "one head per live slot", "inval"),
    (dict(k_cache=T((8, 4, 16, 64))), "same pages", "inval"),
    (dict(k_cache=T((9, 4, 32, 64))), "same pages", "inval"),
    (dict(k_cache=T((9, 4, 16, 64), F16)), "share v's dtype", "inval"),
    (dict(k_cache=None), "require q and k_cache", "inval"),
    (dict(q=T((2, 4, 2, 64))), "(B, U, 1, HD)", "inval"),
    (dict(q=T((3, 4, 1, 64))), "(B, U, 1, HD)", "inval"),
    (dict(out=T((2, 5, 1, 64))), "out must have shape", "inval"),
    (dict(page_table=T((2, 5), I64)), "page_table must be int32", "inval"),
    (dict(page_table=T((3, 5), I32)), "page_table must be int32", "inval"),
    (dict(page_table=T((2, 5), I32, stride=[10, 2])), "unit last stride", "align"),
    (dict(page_table=T((2, 1 << 27), I32)), "2^30 positions", "unsup"),
    (dict(lengths=T((3,), I32)), "lengths must be int32", "inval"),
    (dict(lengths=T((2,), I64)), "lengths must be int32", "inval"),
    (dict(frozen=[0, 0, 3, 0]), "not a head state", "inval"),
    (dict(hidx=[0, 1, 2, 4]), "does not index the 4 compact", "inval"),
    (dict(kvidx=[0, 0, 1, 4]), "must index the HKV heads", "inval"),
    (dict(frozen=[0, 1, 0, 0]), "require patt", "inval"),
    (dict(frozen=[0, 1, 0, 0], patt=T((2, 8, 8), F32), pidx=[0, 2, 0, 0]), "must index patt", "inval"),
    (dict(frozen=[0, 1, 0, 0], patt=T((2, 8, 9), F32), pidx=[0, 1, 0, 0]), "(P, S, S)", "inval"),
    (dict(frozen=[0, 2, 0, 0]), "require alpha/rho/z", "inval"),
    (dict(frozen=[0, 2, 0, 0], alpha=T((4, 8), F32), rho=T((4, 8), F32), z=T((4, 9), F32)), "matching (H, S)", "inval"),
    (dict(frozen=[0, 2, 0, 0], alpha=T((3, 8), F32), rho=T((3, 8), F32), z=T((3, 8), F32)), "matching (H, S)", "inval"),
    (dict(lse=T((2, 4), F32)), "lse must be fp32", "inval"),
    (dict(H=129), "n_heads 129", "unsup"),
    (dict(sm_scale=float("nan")), "sm_scale must be finite", "inval"),
]
STATUS = dict(inval=_ext.SAF_EINVAL, unsup=_ext.SAF_EUNSUPPORTED, align=_ext.SAF_EALIGN)


@pytest.mark.parametrize("kw,msg,status", ATTN_BAD, ids=[str(i) for i in range(len(ATTN_BAD))])
def test_paged_attn_refusals(kw, msg, status):
    L = _ext.lib()
    a, keep = _attn(**kw)
    assert L.saf_paged_attn_fwd(a, None) == STATUS[status]
    assert msg in L.saf_last_error().decode()
    assert L.saf_paged_attn_workspace_bytes(a) == -1


def test_paged_attn_workspace():
    L = _ext.lib()
    a, keep = _attn()
    assert L.saf_paged_attn_workspace_bytes(a) == 0       # 80 positions: one key range
    a, keep = _attn(page_table=T((2, 4096), I32))
    n = L.saf_paged_attn_workspace_bytes(a)
    assert n > 0 and n % 8 == 0
    assert L.saf_paged_attn_fwd(a, None) == _ext.SAF_EWORKSPACE
    a.workspace, a.workspace_bytes = PTR, n - 1
    assert L.saf_paged_attn_fwd(a, None) == _ext.SAF_EWORKSPACE
    a.workspace, a.workspace_bytes = PTR + 4, n
    assert L.saf_paged_attn_fwd(a, None) == _ext.SAF_EALIGN
    a, keep = _attn(q=T((0, 4, 1, 64)), out=T((0, 4, 1, 64)), page_table=T((0, 5), I32), lengths=T((0,), I32))
    assert L.saf_paged_attn_fwd(a, None) == _ext.SAF_OK   # no sequence: nothing to do
    assert L.saf_paged_attn_fwd(None, None) == _ext.SAF_EINVAL


def _append(**kw):
    a = _ext.SafPagedAppendArgs()
    base = dict(q=T((2, 4, 3, 64)), k=T((2, 2, 3, 64)), v=T((2, 2, 3, 64)), q_out=T((2, 4, 3, 64)),
                k_cache=T((9, 2, 16, 64)), v_cache=T((9, 2, 16, 64)), page_table=T((2, 5), I32), positions=T((2,), I32),
                cos=T((80, 64), F32), sin=T((80, 64), F32))
    a.eps = kw.pop("eps", 1e-6)
    base.update(kw)
    for n, t in base.items():
        if t is not None:
            setattr(a, n, t)
    return a


APPEND_BAD = [
    (dict(v=None), "v and v_cache are required", "inval"),
    (dict(v_cache=None), "v and v_cache are required", "inval"),
    (dict(v=T((2, 2, 3, 64), I32)), "unsupported v dtype", "unsup"),
    (dict(v_cache=T((9, 3, 16, 64))), "v's heads", "inval"),
    (dict(v_cache=T((9, 2, 20, 64))), "page size 20", "unsup"),
    (dict(k_cache=None), "k needs k_cache", "inval"),
    (dict(k_cache=T((9, 3, 16, 64))), "k's heads", "inval"),
    (dict(k_cache=T((8, 2, 16, 64))), "k's heads", "inval"),
    (dict(k=T((2, 2, 4, 64))), "k and v batch", "inval"),
    (dict(k=T((2, 2, 3, 64), F16)), "share v's dtype", "inval"),
    (dict(q=T((2, 4, 3, 32))), "q and v batch", "inval"),
    (dict(q_out=None), "q needs q_out", "inval"),
    (dict(q_out=T((2, 5, 3, 64))), "q's shape", "inval"),
    (dict(q=T((2, 4, 3, 64), ptr=PTR + 4)), "not 16-byte aligned", "align"),
    (dict(positions=T((2,), I64)), "positions must be int32", "inval"),
    (dict(counts=T((3,), I32)), "counts must be int32", "inval"),
    (dict(sin=None), "go together", "inval"),
    (dict(sin=T((80, 32), F32)), "one shape", "inval"),
    (dict(cos=T((80, 24), F32), sin=T((80, 24), F32)), "rotary dimension 24", "unsup"),
    (dict(cos=T((80, 128), F32), sin=T((80, 128), F32)), "rotary dimension 128", "unsup"),
    (dict(q_weight=T((64,))), "go together", "inval"),
    (dict(q_weight=T((64,)), k_weight=T((32,))), "k_weight must be", "inval"),
    (dict(q_weight=T((64,)), k_weight=T((64,), F32)), "share a dtype", "inval"),
    (dict(q_weight=T((64,)), k_weight=T((64,)), eps=-1.0), "non-negative", "inval"),
]


@pytest.mark.parametrize("kw,msg,status", APPEND_BAD, ids=[str(i) for i in range(len(APPEND_BAD))])
def test_paged_append_refusals(kw, msg, status):
    L = _ext.lib()
    assert L.saf_paged_append(_append(**kw), None) == STATUS[status]
    assert msg in L.saf_last_error().decode()


def _logp(**kw):
    a = _ext.SafTokenLogprobsArgs()
    a.top, a.scale, a.ignore_index = kw.pop("top", 0), kw.pop("scale", 1.0), -100
    base = dict(logits=T((3, 100)), tokens=T((3,), I64), logp=T((3,), F32), stats=T((3, 2), F32))
    base.update(kw)
    for n, t in base.items():
        if t is not None:
            setattr(a, n, t)
    return a


LOGP_BAD = [
    (dict(logits=T((3, 100), I32)), "unsupported logits dtype", "unsup"),
    (dict(logits=T((300,))), "2-D", "inval"),
    (dict(logits=T((3, 100), stride=[1, 3])), "unit column stride", "align"),
    (dict(tokens=T((4,), I64)), "one entry per row", "inval"),
    (dict(tokens=T((3,), F32)), "int32 or int64", "inval"),
    (dict(logp=None), "logp is required", "inval"),
    (dict(stats=T((3, 3), F32)), "stats must be", "inval"),
    (dict(entropy=T((3,), BF16)), "entropy must be", "inval"),
    (dict(scale=0.0), "positive and finite", "inval"),
    (dict(scale=float("inf")), "positive and finite", "inval"),
    (dict(top=33, top_index=T((3, 33), I64), top_logp=T((3, 33), F32)), "top = 33", "unsup"),
    (dict(top=-1), "top = -1", "unsup"),
    (dict(logits=T((3, 4)), top=5), "top = 5", "unsup"),
    (dict(top=2), "top_index (int64)", "inval"),
    (dict(top=2, top_index=T((3, 2), I32), top_logp=T((3, 2), F32)), "top_index (int64)", "inval"),
]


@pytest.mark.parametrize("kw,msg,status", LOGP_BAD, ids=[str(i) for i in range(len(LOGP_BAD))])
def test_token_logprobs_refusals(kw, msg, status):
    L = _ext.lib()
    a = _logp(**kw)
    assert L.saf_token_logprobs(a, None) == STATUS[status]
    assert msg in L.saf_last_error().decode()
    assert L.saf_token_logprobs_workspace_bytes(a) == -1


def test_token_logprobs_bwd_refusals():
    L = _ext.lib()
    g, d = T((3,), F32), T((3, 100))
    for bad, msg in (((None, None, d), "are required"), ((g, None, None), "are required"),
                     ((T((4,), F32), None, d), "fp32 (R,)"), ((g, g, d), "needs the forward's entropy"),
                     ((g, None, T((3, 99))), "shape and dtype"), ((g, None, T((3, 100), F32)), "shape and dtype"),
                     ((g, None, T((3, 100), stride=[1, 3])), "unit column stride")):
        assert L.saf_token_logprobs_bwd(_logp(), *bad, None) < 0
        assert msg in L.saf_last_error().decode(), msg
    assert L.saf_token_logprobs_bwd(_logp(stats=None), g, None, d, None) < 0
    assert "stats are required" in L.saf_last_error().decode()
    a = _logp(logits=T((1, 200000)), tokens=T((1,), I64), logp=T((1,), F32), stats=T((1, 2), F32))
    assert L.saf_token_logprobs_workspace_bytes(a) > 0
    assert L.saf_token_logprobs(a, None) == _ext.SAF_EWORKSPACE


def test_struct_layouts(tmp_path):
    """The ctypes blocks match the header (as test_abi_layout.py does for the
    prefill's)."""
    import ctypes
    import shutil
    from test_abi_layout import _c_layout
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    for cname, cls in (("saf_paged_append_args", _ext.SafPagedAppendArgs), ("saf_paged_attn_args", _ext.SafPagedAttnArgs),
                       ("saf_token_logprobs_args", _ext.SafTokenLogprobsArgs)):
        names = [f[0] for f in cls._fields_]
        c = _c_layout(tmp_path, cname, names)
        assert c["__sizeof"] == ctypes.sizeof(cls)
        for n in names:
            assert c[n] == getattr(cls, n).offset, (cname, n)


def test_cpu_tensors_and_python_checks():
    kc = torch.zeros(3, 2, 16, 64)
    table, one = torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    frozen = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 64)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        kernel.paged_mixed_attn(x, kc, kc, table, one, None, frozen)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        kernel.paged_append_(x, x, kc, kc, table, one)
    with pytest.raises(RuntimeError, match="HIP devices only"):
        kernel.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError, match="leading shape"):
        kernel.token_logprobs(torch.zeros(2, 5), torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="go together"):
        kernel.paged_append_(x, x, None, kc, table, one)
    with pytest.raises(ValueError, match="go together"):
        kernel.paged_append_(x, x, kc, kc, table, one, cos=torch.zeros(5, 64))
