"""The token after the prefill: a paged key / value cache and its attention.

``fused_mixed_attn`` runs whole sequences.  These two operators continue them
one token at a time, with the same head states (live, dense-frozen,
decomposed-frozen), compact live slots and GQA map:

    q = paged_append_(k, v, k_cache, v_cache, page_table, positions, q=q, cos=cos, sin=sin)
    y = paged_mixed_attn(q, k_cache, v_cache, page_table, lengths, patt, frozen, hidx, ...)

A cache is a pool of pages: ``k_cache`` (P, U, PS, HD) for the live heads' U
compact slots and ``v_cache`` (P, H, PS, HD) for every head (with ``kvidx``
both hold the HKV raw heads; frozen heads never read keys), PS token slots a
page (a power of two, at least 16).  ``page_table`` (B, N) int32 lists each
sequence's pages: its position s is slot s % PS of page
``page_table[b, s // PS]``.  Page ids, positions and lengths are device data
that no call reads back; what they get wrong shows as NaN, never as a stray
access (libsafattn.so ``saf_paged_append``, ``saf_paged_attn_fwd``).  Without
derivatives: tensors that need a gradient or carry a tangent are refused.
"""
import ctypes

import torch

from . import _ext
from .fused_attn import _table, decomposed_logz

_stream = torch._C._cuda_getCurrentRawStream
_APPEND = ("v", "k", "q", "q_out", "k_cache", "v_cache", "page_table", "positions", "counts", "cos", "sin")
_APPEND_AT = _ext.offsets(_ext.SafPagedAppendArgs, *_APPEND)
_WEIGHTS_AT = _ext.offsets(_ext.SafPagedAppendArgs, "q_weight", "k_weight")
_ATTN_AT = _ext.offsets(_ext.SafPagedAttnArgs, "q", "k_cache", "v_cache", "out", "lse", "patt", "alpha", "rho", "z",
                        "page_table", "lengths")


def _rows_of(t):
    """A cos / sin cache without its leading singleton dims."""
    if t.dim() > 2 and t.numel() != t.size(-2) * t.size(-1):
        raise ValueError(f"cos and sin must be (T', RD) caches, with leading singleton dims at most (got {tuple(t.shape)})")
    return t.reshape(t.shape[-2:])


def paged_append_(k, v, k_cache, v_cache, page_table, positions, counts=None, q=None, cos=None, sin=None,
                  q_weight=None, k_weight=None, eps=1e-6):
    """Write T new tokens per sequence into the caches, in place, rotating
    them to their positions; returns the rotated q (None without q).

      k        (B, U, T, HD) keys of the live slots (the HKV heads with GQA),
               None when no head is live (k_cache None as well)
      v        (B, H, T, HD) values of every head (the HKV heads with GQA)
      positions (B,) int32, the position of each sequence's first new token
      counts   (B,) int32, new tokens per sequence (right-padded batches);
               default T.  The rest of a sequence writes nothing and its rows
               of the returned q are zero
      q        (B, UQ, T, HD) queries, not modified
      cos, sin (T', RD) caches (leading singleton dims are dropped), row s for
               position s: Llama half rotation of the first RD <= HD elements
               (a multiple of 16); None: no rotation
      q_weight, k_weight  (HD,) per-head RMSNorm weights, applied before the
               rotation: w x / sqrt(mean(x^2) + eps)
    fp32 arithmetic, one rounding.  A token whose position lies outside the
    page table or the cos / sin caches, or whose page id is not a page of the
    caches, is not written, and its rows of q are NaN."""
    if (k is None) != (k_cache is None):
        raise ValueError("k and k_cache go together")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    dev = _ext.device_index("paged_append_", v)
    out = None
    if q is not None:
        # token-major like the projection it came from, so that a token's rows
        # follow each other
        B, U, T, HD = q.shape
        out = torch.empty_strided((B, U, T, HD), (T * U * HD, HD, U * HD, 1), device=v.device, dtype=q.dtype)
        if U == 0:
            q = None
    if v.numel() == 0 and v.dim() == 4 and v.size(1) and v.size(3):
        return out   # no sequence or no token
    if k is not None and k.size(1) == 0:
        k = k_cache = None
    if cos is not None and (cos.dim() != 2 or sin.dim() != 2):
        cos, sin = _rows_of(cos), _rows_of(sin)
    args = _ext.SafPagedAppendArgs()
    block, fill = ctypes.addressof(args), _ext.bind().fill
    tensors = (v, k, q, None if q is None else out, k_cache, v_cache, page_table, positions, counts, cos, sin)
    held = None
    mask = fill("paged_append_", block, _APPEND_AT, 7, dev, True, *tensors)
    if mask:
        held = _ext.aligned_copies("paged_append_", block, _APPEND_AT, mask, dev, tensors)  # noqa: F841
    if q_weight is not None or k_weight is not None:  # module parameters, which may need gradients elsewhere
        fill("paged_append_", block, _WEIGHTS_AT, 0, dev, False, q_weight, k_weight)
    args.eps = eps
    with _ext.on_device(dev):
        rc = _ext.lib().saf_paged_append(args, _stream(dev))
    if rc:
        _ext.check(rc)
    return out


def paged_mixed_attn(q, k_cache, v_cache, page_table, lengths, patt, frozen, hidx=None, pidx=None, sm_scale=None,
                     alpha=None, rho=None, z=None, validate=True, kvidx=None, lse=None):
    """Attention of the newest token of each sequence over its cached tokens,
    all heads in one call.

      q        (B, U, 1, HD) compact live-head queries
      k_cache, v_cache, page_table   see the module's docstring
      lengths  (B,) int32 cached tokens, the newest included: the query stands
               at position i = lengths - 1.  0 gives zero rows (an idle slot
               of a batch)
      patt, frozen, hidx, pidx, sm_scale, alpha, rho, z, kvidx, lse
               as in fused_mixed_attn: row i of the patterns (closed-form
               heads through their alpha / rho / z); lse (B, H, 1) fp32
    Returns (B, H, 1, HD).  A length past the page table, a page id outside
    the caches, and for a frozen head a length past its pattern give NaN rows.
    validate also checks shapes with the reference operator's messages."""
    dev = _ext.device_index("paged_mixed_attn", v_cache)
    if sm_scale is None:
        sm_scale = v_cache.size(-1) ** -0.5
    if alpha is not None and z is None:
        z = decomposed_logz(alpha.float(), rho.float())
    frozen_h, frozen_c = _table(frozen)
    if validate:
        _validate(q, k_cache, v_cache, page_table, lengths, patt, frozen_h, alpha, rho, z, kvidx)
    H = len(frozen_c)
    args = _ext.SafPagedAttnArgs()
    args.frozen = frozen_c
    for name, t in (("hidx", hidx), ("pidx", pidx), ("kvidx", kvidx)):
        if t is not None:
            c = _table(t)[1]
            if len(c) < H:
                raise ValueError(f"{name} must have one entry per output head")
            setattr(args, name, c)
    B = page_table.size(0)
    out = torch.empty((B, H, 1, v_cache.size(-1)), device=v_cache.device, dtype=v_cache.dtype)
    if B == 0:
        return out
    if q is None or q.numel() == 0:
        q = k_cache = None
    block = ctypes.addressof(args)
    tensors = (q, k_cache, v_cache, out, lse, patt, alpha, rho, z, page_table, lengths)
    held = None
    mask = _ext.bind().fill("paged_mixed_attn", block, _ATTN_AT, 1, dev, True, *tensors)
    if mask:
        held = _ext.aligned_copies("paged_mixed_attn", block, _ATTN_AT, mask, dev, tensors)  # noqa: F841
    args.n_heads = H
    args.sm_scale = sm_scale
    L = _ext.lib()
    with _ext.on_device(dev):
        nbytes = L.saf_paged_attn_workspace_bytes(args)
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=v_cache.device)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
        rc = L.saf_paged_attn_fwd(args, _stream(dev))
    if rc:
        _ext.check(rc)
    return out


def _validate(q, k_cache, v_cache, page_table, lengths, patt, frozen, alpha, rho, z, kvidx):
    assert v_cache.ndim == 4 and page_table.ndim == 2 and lengths.ndim == 1, \
        "v_cache must be (P, H, PS, HD), page_table (B, N) and lengths (B,)"
    assert page_table.dtype == lengths.dtype == torch.int32, "page_table and lengths must be int32"
    B = page_table.size(0)
    assert lengths.size(0) == B, "lengths must have one entry per sequence"
    if kvidx is None:
        assert v_cache.size(1) == len(frozen), "v_cache must hold one head per output head (or pass kvidx)"
    if (frozen == 0).any():
        assert q is not None and k_cache is not None, "live heads require q and k_cache"
        assert q.ndim == 4 and q.shape[0] == B and q.shape[2] == 1 and q.shape[3] == v_cache.size(3), \
            "q must be (B, U, 1, HD): one new token per sequence"
    assert patt is not None or not (frozen == 1).any(), "dense-frozen heads require patt"
    if (frozen == 2).any():
        assert alpha is not None and rho is not None and alpha.shape == rho.shape == z.shape, \
            "alpha, rho, and z must have matching (H, S) shapes"
        assert alpha.shape[0] == len(frozen), "decomposed buffers must have shape (H, S)"
