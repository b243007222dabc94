"""Activations in 8 bits between the forward and the backward pass.

A training step keeps what its backward pass reads; most of that are the MLP's
activations (nanogpt/model.py:1193-1207).  ``pack_activation`` holds a tensor as
int8 multiples of a power-of-two step per 32 channels (libsafattn.so
``saf_act_pack``): 1.03 bytes an element, off by at most 1/128 of its block's
largest magnitude.  ``gelu_packed`` is nn.GELU() that keeps its input so, and
``mlp_packed`` a whole MLP that keeps its two activations so: 5.2 C bytes a
token for the (C, 4 C) MLP of the GPT, where the autograd of bf16 tensors keeps 18 C.
The forward pass is computed from the exact values; the gradients see the held
ones.
"""
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _ext
from .indexed_linear import _compute_args


class PackedActivation(NamedTuple):
    q: torch.Tensor      # (..., C) int8 multiples of the step
    exp: torch.Tensor    # (..., ceil(C / 32)) uint8: step 2^(exp - 127); 255: the block was not finite
    dtype: torch.dtype   # of the activation


def pack_activation(x):
    """x (..., C) in 8 bits.  For a block of 32 channels (a row's last one may be
    short) with the largest magnitude m the step is 2^(floor(log2 m) - 6), and each
    value its nearest multiple (half to even), at most 127 steps.  A block with an
    infinity or NaN comes back as NaN.  Without derivative (the result is what a
    backward pass keeps): an x that needs a gradient is refused while grad mode is on."""
    return PackedActivation(*_ext.bind().pack_activation(x), x.dtype)


def unpack_activation(p, dtype=None):
    """The activation that p stands for, in p's dtype (exact) or another of
    float32, bfloat16 and float16 (rounded once)."""
    return _ext.bind().unpack_activation(p.q, p.exp, _ext.dtype_code("unpack_activation", p.dtype if dtype is None else dtype))


def gelu_packed(x):
    """Exact GELU of x (..., C), float32, bfloat16 or float16.  Its backward is
    dy (Phi(h) + h phi(h)) for the 8-bit h of x (see pack_activation), which is
    all that it keeps (reverse mode, once); without a gradient nothing is packed."""
    return _ext.bind().gelu_packed(x, False)


class _MlpPacked(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w_fc, w_proj, b_fc, b_proj):
        bind = _ext.bind()
        y, q, e = bind.gelu_packed(F.linear(x, w_fc, b_fc), True)
        ctx.save_for_backward(*(bind.pack_activation(x) if w_fc.requires_grad else (None, None)), q, e, w_fc, w_proj)
        return F.linear(y, w_proj, b_proj)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        bind = _ext.bind()
        xq, xe, q, e, w_fc, w_proj = ctx.saved_tensors
        need_x, need_fc, need_proj, need_bfc, need_bproj = ctx.needs_input_grad
        g = gy.reshape(-1, gy.size(-1))
        dx = dw_fc = dw_proj = db_fc = db_proj = None
        # sums over the rows as products: a reduction's own kernels would not
        # take a capture
        ones = g.new_ones(1, g.size(0)) if need_bfc or need_bproj else None
        if need_bproj:
            db_proj = (ones @ g).view(-1)
        if need_x or need_fc or need_bfc or need_proj:
            du, act = bind.gelu_packed_bwd(q, e, (g @ w_proj).view(q.shape), need_proj)
            if need_proj:
                dw_proj = g.t() @ act.view(-1, act.size(-1))
                del act
            du = du.view(-1, du.size(-1))
            if need_bfc:
                db_fc = (ones @ du).view(-1)
            if need_fc:
                x = bind.unpack_activation(xq, xe, _ext.dtype_code("mlp_packed", g.dtype))
                dw_fc = du.t() @ x.view(-1, x.size(-1))
            if need_x:
                dx = (du @ w_fc).view(xq.shape if xq is not None else (*gy.shape[:-1], w_fc.size(1)))
        return dx, dw_fc, dw_proj, db_fc, db_proj


def mlp_packed(x, w_fc, w_proj, b_fc=None, b_proj=None):
    """gelu(x @ w_fc.T + b_fc) @ w_proj.T + b_proj for x (..., C), w_fc (F, C) and
    w_proj (C', F), all of one dtype (under autocast they are cast to its); exact
    GELU.  Keeps x and the GELU's input in 8 bits and recomputes the GELU's output
    from them; the gradients of x, the weights and the biases are those of the
    held activations (reverse mode, once).  Without a gradient nothing is packed.  The
    products are library GEMMs."""
    x, (w_fc, w_proj, b_fc, b_proj) = _compute_args(x, [w_fc, w_proj, b_fc, b_proj])
    if w_fc.dim() != 2 or w_proj.dim() != 2 or x.size(-1) != w_fc.size(1) or w_proj.size(1) != w_fc.size(0):
        raise ValueError(f"mlp_packed takes x (..., C), w_fc (F, C) and w_proj (C', F) (got {tuple(x.shape)}, "
                         f"{tuple(w_fc.shape)} and {tuple(w_proj.shape)})")
    if any(t is not None and t.dtype != x.dtype for t in (w_fc, w_proj, b_fc, b_proj)):
        raise ValueError("mlp_packed takes tensors of one dtype")
    _ext.bind().check_differentiable("mlp_packed", x, w_fc, w_proj, b_fc, b_proj)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in (x, w_fc, w_proj, b_fc, b_proj)):
        return F.linear(gelu_packed(F.linear(x, w_fc, b_fc)), w_proj, b_proj)
    return _MlpPacked.apply(x, w_fc, w_proj, b_fc, b_proj)
