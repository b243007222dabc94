"""Log probabilities of given tokens: what a model answers with, and its loss.

``token_logprobs`` reads each row of logits once and gives the log probability
of the row's token, the entropy of the distribution and its most likely
alternatives (libsafattn.so ``saf_token_logprobs``); its backward writes the
logits' gradient in one pass (``saf_token_logprobs_bwd``), so
``-token_logprobs(logits, tokens).logp.mean()`` is the cross-entropy loss.  It
serves the evaluation that the reference does with log_softmax and gather
(/root/reference/nanogpt/eval_nanogpt_logprobs.py) and sampling loops that
report alternatives.
"""
import ctypes
from typing import NamedTuple, Optional

import torch

from . import _ext

_stream = torch._C._cuda_getCurrentRawStream
_AT = _ext.offsets(_ext.SafTokenLogprobsArgs, "logits", "tokens", "logp", "entropy", "stats", "top_index", "top_logp")
_GRAD_AT = tuple(i * ctypes.sizeof(_ext.SafTensor) for i in range(3))


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor                  # (...) fp32
    entropy: Optional[torch.Tensor]     # (...) fp32, nats
    top_index: Optional[torch.Tensor]   # (..., top) int64
    top_logp: Optional[torch.Tensor]    # (..., top) fp32


def _forward(logits, tokens, top, entropy, scale, ignore_index, keep_stats):
    R, dev = logits.size(0), logits.device
    f32 = dict(device=dev, dtype=torch.float32)
    logp = torch.empty(R, **f32)
    stats = torch.empty(R, 2, **f32) if keep_stats else None
    ent = torch.empty(R, **f32) if entropy else None
    idx = torch.empty(R, top, device=dev, dtype=torch.int64) if top else None
    tlp = torch.empty(R, top, **f32) if top else None
    args = _ext.SafTokenLogprobsArgs()
    index = logits.get_device()
    _ext.desc_fill()("token_logprobs", ctypes.addressof(args), _AT, 0, index, False, logits, tokens, logp, ent, stats, idx,
                     tlp)
    args.top, args.ignore_index, args.scale = top, ignore_index, scale
    L = _ext.lib()
    with _ext.on_device(index):
        nbytes = L.saf_token_logprobs_workspace_bytes(args)
        if nbytes > 0:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
        rc = L.saf_token_logprobs(args, _stream(index))
    if rc:
        _ext.check(rc)
    return logp, ent, idx, tlp, stats


class _TokenLogprobsFn(torch.autograd.Function):

    @staticmethod
    def forward(ctx, logits, tokens, top, entropy, scale, ignore_index):
        logp, ent, idx, tlp, stats = _forward(logits, tokens, top, entropy, scale, ignore_index, True)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.scale, ctx.ignore_index = scale, ignore_index
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(idx, tlp)
        return logp, ent, idx, tlp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, glogp, gent, _gi, _gt):
        logits, tokens, stats, ent = ctx.saved_tensors
        if glogp is None and gent is None:
            return (None,) * 6
        glogp = torch.zeros_like(stats[:, 0]) if glogp is None else glogp.float()
        gent = None if gent is None else gent.float()
        R, V = logits.shape
        dx = torch.empty(R, V, device=logits.device, dtype=logits.dtype)
        args = _ext.SafTokenLogprobsArgs()
        index, fill = logits.get_device(), _ext.desc_fill()
        fill("token_logprobs", ctypes.addressof(args), _AT, 0, index, False, logits, tokens, None, ent, stats, None, None)
        args.ignore_index, args.scale = ctx.ignore_index, ctx.scale
        descs = (_ext.SafTensor * 3)()
        fill("token_logprobs", ctypes.addressof(descs), _GRAD_AT, 0, index, False, glogp, gent, dx)
        with _ext.on_device(index):
            rc = _ext.lib().saf_token_logprobs_bwd(args, descs[0], descs[1], descs[2], _stream(index))
        if rc:
            _ext.check(rc)
        return dx, None, None, None, None, None


def _leaf_edge(logits):
    """The gradient edge of logits that are a leaf (None otherwise), kept alive
    by the caller while the autograd graph is built; raises in a graph capture
    where an eager graph of this operator still holds the leaf.

    The leaf's node belongs to the stream of the call that made it.  A captured
    backward would make that stream wait for the capturing one, and with it
    join the capture without ever leaving it: torch ends the process there."""
    if logits.grad_fn is not None:
        return None
    edge = torch.autograd.graph.get_gradient_edge(logits)
    stream = _ext.current_stream_ptr(logits.device)
    if edge.node.metadata.setdefault("saf_stream", stream) != stream and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("token_logprobs: an eager autograd graph of these logits, made on another stream, is still "
                           "alive; release it before capturing their gradient")
    return edge


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
    to the logits is rounded once to their dtype.  As with log_softmax, a row
    holding NaN or +inf, or nothing above -inf, gives NaN (its top indices are
    then some indices of the row)."""
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must have the logits' leading shape (got {tuple(tokens.shape)} for "
                         f"{tuple(logits.shape)})")
    _ext.device_index("token_logprobs", logits)
    top, scale = int(top), float(scale)
    x, t = logits, tokens
    if x.dim() != 2:
        x, t = x.reshape(-1, x.size(-1)), t.reshape(-1)
    if x.stride(1) != 1 and x.size(1) > 1:
        x = x.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        edge = _leaf_edge(logits)  # noqa: F841  (alive until the graph holds it)
        logp, ent, idx, tlp = _TokenLogprobsFn.apply(x, t, top, bool(entropy), scale, int(ignore_index))
    else:
        logp, ent, idx, tlp, _ = _forward(x, t, top, entropy, scale, int(ignore_index), False)
    if logits.dim() != 2:
        lead = tokens.shape
        logp = logp.view(lead)
        ent = None if ent is None else ent.view(lead)
        idx, tlp = (None, None) if idx is None else (idx.view(*lead, top), tlp.view(*lead, top))
    return TokenLogprobs(logp, ent, idx, tlp)
