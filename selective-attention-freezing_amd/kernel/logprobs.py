"""Log probabilities of given tokens: what a model answers with, and its loss.

``token_logprobs`` reads each row of logits once and gives the log probability
of the row's token, the entropy of the distribution and its most likely
alternatives (libsafattn.so ``saf_token_logprobs``); its backward writes the
logits' gradient in one pass (``saf_token_logprobs_bwd``), so
``-token_logprobs(logits, tokens).logp.mean()`` is the cross-entropy loss.  It
serves the evaluation that the reference does with log_softmax and gather
(nanogpt/eval_nanogpt_logprobs.py) and sampling loops that
report alternatives.
"""
from typing import NamedTuple, Optional

import torch

from . import _ext


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                  # (...) fp32
    entropy: Optional[torch.Tensor]     # (...) fp32, nats
    top_index: Optional[torch.Tensor]   # (..., top) int64
    top_logp: Optional[torch.Tensor]    # (..., top) fp32


def token_logprobs(logits, tokens, top=0, entropy=False, scale=1.0, ignore_index=-100):
    """Log probabilities of ``tokens`` (...) under softmax(scale * logits)
    for logits (..., V) in float32, bfloat16 or float16.

      tokens   int64 or int32 indices; ``ignore_index`` marks rows whose logp
               is 0 and which get no gradient through it; any other index
               outside 0..V-1 gives NaN
      top      alternatives per row (0..32): the indices and log probabilities
               of the largest logits, equal ones by lower index.  Not
               differentiable
      entropy  also return -sum p log p (nats)
      scale    1 / temperature, > 0
    fp32 arithmetic throughout; the gradient of logp and entropy with respect
    to the logits is rounded once to their dtype (reverse mode, once; logits with
    a forward-mode tangent are refused).  As with log_softmax, a row
    holding NaN or +inf, or nothing above -inf, gives NaN (its top indices are
    then some indices of the row)."""
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must have the logits' leading shape (got {tuple(tokens.shape)} for "
                         f"{tuple(logits.shape)})")
    _ext.device_index("token_logprobs", logits)
    top = int(top)
    x, t = logits, tokens
    if x.dim() != 2:
        x, t = x.reshape(-1, x.size(-1)), t.reshape(-1)
    if x.stride(1) != 1 and x.size(1) > 1:
        x = x.contiguous()
    logp, ent, idx, tlp = _ext.bind().token_logprobs(x, t, top, entropy, float(scale), int(ignore_index))
    if logits.dim() != 2:
        lead = tokens.shape
        logp = logp.view(lead)
        ent = None if ent is None else ent.view(lead)
        idx, tlp = (None, None) if idx is None else (idx.view(*lead, top), tlp.view(*lead, top))
    return TokenLogprobs(logp, ent, idx, tlp)
