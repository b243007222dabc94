"""Captured decoding steps against eager ones while the rest of the program
goes on: other prefills, changed parameters, memory in use again."""
import pytest
import torch

from nanogpt import decode
from test_model import _small_model

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _capture(m, tok, cache, before=lambda: None):
    """decode_tokens as a graph, behind a warm-up on another cache and before()."""
    warm = decode.PagedCache(m, cache.lengths.numel(), page_size=16)
    decode.prefill(m, tok[:, None].clone(), warm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.reserve(1)
        decode.decode_tokens(m, tok, warm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    before()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = decode.decode_tokens(m, tok, cache)
    return graph, logits


def _junk():
    """Whatever the allocator has free, in use with other values."""
    return [torch.full((n,), 9e3, device="cuda") for n in (1 << 9, 1536, 1 << 11, 1 << 14, 1 << 17, 1 << 19, 1 << 21)
            for _ in range(4)]


def _replays(m, x, at, n, graph, logits, tok, cache, twin):
    for i in range(at, at + n):
        tok.copy_(x[0, i:i + 1])
        want = decode.decode_step(m, x[0, i:i + 1], twin)
        torch.cuda.synchronize()
        cache.reserve(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want), i


@pytest.mark.parametrize("warm", [False, True])
def test_trainable_patterns(warm):
    """The step's row normalisers outlive a prefill of another width, and
    follow the parameters once the cache was checked."""
    import supplement
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    supplement.enable(m)
    with torch.no_grad():
        twin, cache = decode.PagedCache(m, 1, page_size=16), decode.PagedCache(m, 1, page_size=16)
        decode.prefill(m, x[:, :60], twin)
        decode.prefill(m, x[:, :60], cache)
        tok = x[0, 60:61].clone()
        forget = m._saf_patterns._step_z.clear    # the capture finds no normalisers
        graph, logits = _capture(m, tok, cache, (lambda: None) if warm else forget)
        decode.prefill(m, x[:, :37], decode.PagedCache(m, 1, page_size=16))
        held = _junk()
        _replays(m, x, 60, 4, graph, logits, tok, cache, twin)
        m.transformer.h[0].attn.dyn_alpha[3, :20] += 0.5
        m._saf_patterns.invalidate()
        cache.check(m)
        _replays(m, x, 64, 3, graph, logits, tok, cache, twin)
        assert len(held) > 0


@pytest.mark.parametrize("bias", [False, True])
def test_packed_weights(bias):
    """eval() again and a prefill, which packs the projection weights anew,
    leave the captured step's rows in place; so does a change of the weights,
    which the step follows."""
    if bias:
        from test_gpu_decode import _plain_model
        m = _plain_model(bias=True, frozen=(1,))
        x = torch.randint(0, 512, (1, 128), generator=torch.Generator().manual_seed(3)).cuda()
    else:
        m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    with torch.no_grad():
        twin, cache = decode.PagedCache(m, 1, page_size=16), decode.PagedCache(m, 1, page_size=16)
        decode.prefill(m, x[:, :60], twin)
        decode.prefill(m, x[:, :60], cache)
        tok = x[0, 60:61].clone()
        graph, logits = _capture(m, tok, cache)
        _replays(m, x, 60, 2, graph, logits, tok, cache, twin)
        m.train()
        m.eval()
        decode.prefill(m, x[:, :37], decode.PagedCache(m, 1, page_size=16))
        held = _junk()
        _replays(m, x, 62, 2, graph, logits, tok, cache, twin)
        m.transformer.h[1].attn.v_proj.weight.mul_(1.5)
        cache.check(m)
        _replays(m, x, 64, 2, graph, logits, tok, cache, twin)
        assert len(held) > 0
