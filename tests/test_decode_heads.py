"""Changed live heads and a wrong number of tokens are noticed by every call on a
cache, the capturable half of a step among them (CPU), and changed heads are
refused inside a capture."""
import pytest
import torch

from nanogpt import decode
from test_decode_cache import _model


def _swap(attn):
    """As many live heads, but others."""
    attn.dyn_frozen[1], attn.dyn_frozen[2] = False, True
    attn.dyn_pattern_slot[2], attn.dyn_pattern_slot[1] = int(attn.dyn_pattern_slot[1]), -1
    attn._fz_dirty = True


def _frozen_model(device="cpu"):
    m = _model().to(device)
    for blk in m.transformer.h:
        blk.attn.freeze_heads([1], torch.rand(1, 64, 64, device=device))
    return m


@pytest.mark.parametrize("refreshed", [False, True])
@pytest.mark.parametrize("call", ["decode_tokens", "decode_step", "prefill", "check"])
def test_every_call_checks(call, refreshed):
    m = _frozen_model()
    cache = decode.PagedCache(m, 1, page_size=16)
    _swap(m.transformer.h[1].attn)
    if refreshed:
        m.transformer.h[1].attn._refresh_freeze_cache()
    calls = dict(decode_tokens=lambda: decode.decode_tokens(m, torch.tensor([1]), cache),
                 decode_step=lambda: decode.decode_step(m, torch.tensor([1]), cache),
                 prefill=lambda: decode.prefill(m, torch.zeros(1, 5, dtype=torch.long), cache),
                 check=lambda: cache.check(m))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="live heads changed"):
            calls[call]()
        assert cache._held == [0]


@pytest.mark.parametrize("call", [decode.decode_tokens, decode.decode_step])
@pytest.mark.parametrize("n", [0, 1, 2, 6])
def test_one_token_per_sequence(call, n):
    """A single token is not spread over the batch."""
    m = _frozen_model()
    cache = decode.PagedCache(m, 3, page_size=16)
    with pytest.raises(ValueError, match="one token per sequence"):
        call(m, torch.zeros(n, dtype=torch.long), cache)
    assert cache._held == [0, 0, 0]


@pytest.mark.gpu
def test_captures_are_refused():
    """Before anything of the step is recorded."""
    m = _frozen_model("cuda").bfloat16()
    cache = decode.PagedCache(m, 1, page_size=16)
    x = torch.zeros(1, 5, dtype=torch.long, device="cuda")
    decode.prefill(m, x, cache)
    decode.decode_step(m, x[:, 0], cache)
    cache.reserve(1)
    for swap in (lambda attn: None, _swap):
        attn = m.transformer.h[1].attn
        swap(attn)
        attn._fz_dirty = True
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                decode.decode_tokens(m, x[:, 0], cache)
        torch.cuda.synchronize()
        if swap is not _swap:
            cache.check(m)                        # the same heads: good again
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                decode.decode_tokens(m, x[:, 0], cache)
        else:
            with pytest.raises(RuntimeError, match="live heads changed"):
                cache.check(m)
