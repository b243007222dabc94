"""Embedding rows by token, and the embedding's gradient.

``embed_tokens`` is the lookup that starts a forward pass (nn.Embedding of the
reference's GPT, nanogpt/model.py:1312-1417), with a factor and the activations'
own dtype (libsafattn.so ``saf_embed_fwd``); its backward sorts the tokens and
writes the whole gradient once, the rows of each word added in an order that the
tokens and the shape alone decide (``saf_embed_bwd``), so it is the same in every
run, where a scatter with atomics is not.
"""
from . import _ext


def embed_tokens(tokens, weight, scale=1.0, ignore_index=-100, dtype=None):
    """scale * weight[tokens] for tokens (...) int64 or int32 and weight (V, C) in
    float32, bfloat16 or float16; returns (..., C).

      ignore_index  tokens of padding: zero rows without a gradient.  Any other
                    token outside 0..V-1 gives a NaN row, without a gradient
                    either (tokens are device data that no call reads back)
      dtype         of the result; default the weight's.  float32 and one 16-bit
                    type may meet in either direction, bfloat16 and float16 not
    fp32 arithmetic, one rounding.  Differentiable in weight (reverse mode, once):
    the gradient is dense, in the weight's dtype."""
    return _ext.bind().embed_tokens(tokens, weight, float(scale), int(ignore_index),
                                    _ext.dtype_code("embed_tokens", dtype))
