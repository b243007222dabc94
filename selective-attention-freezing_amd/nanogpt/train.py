"""A training pass of the GPT of ``nanogpt.model`` on the framework's own operators
around its products and attention.

    logp = token_logprobs(model, idx, targets).logp      # (B, T)
    (-logp.mean()).backward()

computes what ``GPT.token_logprobs`` does, with ``kernel.embed_tokens`` for the
embedding, each residual addition fused with the LayerNorm behind it
(``kernel.add_layernorm``), and the MLPs' activations kept in 8 bits for the
backward pass (``kernel.mlp_packed``; ``packed=False`` keeps them whole).  Under
autocast the residual stream has the weights' float32 and the branches the
autocast dtype.  An embedding, block, norm or MLP that is not the model's own, or
has hooks, other options, another activation or adapted projections, is called as
it is, and so are the model's own methods where a subclass has other ones.
"""
import torch
import torch.nn as nn

import kernel as _kernel_mod
from kernel import _ext
from nanogpt.model import GPT, MLP, Block, LayerNorm


def forward_hidden(model, idx, packed=True):
    """Hidden states (B, T, C) of every position behind the last norm,
    differentiable in every parameter of the model that the tokens reach.  A token
    outside the vocabulary, -100 included, makes its sequence NaN."""
    T = idx.size(1)
    if T > model.config.block_size:
        raise ValueError(f"sequences of {T} tokens exceed the model's block size {model.config.block_size}")
    if torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        # weights of torch's own operators as well, which would not refuse the capture
        _ext.bind().check_differentiable("nanogpt.train", *model.parameters())
    x, rope = model.prepare_inputs(idx) if _own(model, "prepare_inputs") else _inputs(model, idx)
    dtype = _branch_dtype(x)
    tr = model.transformer
    d = None                                     # what is not yet added to the residual
    for block in tr.h:
        if not _stock(block, Block):
            x, d = block(x if d is None else x + d, rope=rope), None
            continue
        x, h = _norm(block.ln_1, x, d, dtype)
        x, h = _norm(block.ln_2, x, block.attn(h, rope=rope), dtype)
        d = _mlp(block.mlp, h, packed)
    return _norm(tr.ln_f, x, d, dtype)[1]


def _stock(module, kind):
    """Whether calling module computes kind's forward and nothing else: no subclass, no
    forward of the instance's own, no hooks."""
    return (type(module) is kind and "forward" not in vars(module)
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


def _own(model, name):
    """Whether a model has a method of its own in place of GPT's."""
    return name in vars(model) or getattr(type(model), name, None) not in (None, getattr(GPT, name))


def _branch_dtype(x):
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


def _inputs(model, idx):
    """GPT.prepare_inputs on embed_tokens."""
    tr, T = model.transformer, idx.size(1)
    x = _embed(tr.wte, idx)
    if model.rotary is None:
        return x + tr.wpe(torch.arange(T, device=idx.device)), None
    return x, model.rotary(T, _branch_dtype(x))


def _embed(wte, idx):
    if not _stock(wte, nn.Embedding) or wte.padding_idx is not None or wte.max_norm is not None \
            or wte.scale_grad_by_freq or wte.sparse:
        return wte(idx)
    # no token of a batch is padding: one outside the vocabulary gives NaNs, not zeros
    return _kernel_mod.embed_tokens(idx, wte.weight, ignore_index=-2 ** 63)


def _norm(ln, x, d, dtype):
    """(x + d, ln of it); without d the norm of x in dtype."""
    fused = _stock(ln, LayerNorm)
    # a sum of one shape, and of x's type
    if d is not None and not (fused and d.shape == x.shape and torch.promote_types(x.dtype, d.dtype) == x.dtype):
        x, d = x + d, None
    if not fused:
        return x, ln(x)
    return _kernel_mod.add_layernorm(x, d, ln.weight, ln.bias, dtype=dtype if d is None else None)


def _mlp(mlp, h, packed):
    if not (packed and _stock(mlp, MLP) and _stock(mlp.c_fc, nn.Linear) and _stock(mlp.c_proj, nn.Linear)
            and _stock(mlp.gelu, nn.GELU) and mlp.gelu.approximate == "none"):
        return mlp(h)
    return _kernel_mod.mlp_packed(h, mlp.c_fc.weight, mlp.c_proj.weight, mlp.c_fc.bias, mlp.c_proj.bias)


def token_logprobs(model, idx, tokens, packed=True, **kw):
    """Log probabilities of tokens (B, T) as the next tokens of idx (B, T), with
    kernel.token_logprobs' options; -logp.mean() is the training loss."""
    if _own(model, "forward_all_positions"):
        logits = model.forward_all_positions(idx)
    else:
        logits = model.lm_head(model.forward_hidden(idx) if _own(model, "forward_hidden") else forward_hidden(model, idx, packed))
    return _kernel_mod.token_logprobs(logits, tokens, **kw)
