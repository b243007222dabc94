"""nanogpt.decode after a call that raised: the cache is as it was (CPU, where
the model raises at its first operator; and a failing layer on the device)."""
import pytest
import torch

from nanogpt import decode
from test_decode_cache import _model


def _state(cache):
    return (list(cache._held), list(cache._on), [list(p) for p in cache._pages], sorted(cache._free),
            cache.page_table.tolist(), cache.lengths.tolist(), cache.active.tolist())


@pytest.mark.parametrize("width,counts,error", [(65, [64, 3], ValueError), (65, None, ValueError), (40, None, RuntimeError),
                                                (40, [40, 17], RuntimeError)])
def test_prefill_that_raises(width, counts, error):
    """Too wide for the model with counts that fit, and a forward that fails."""
    m = _model()
    cache = decode.PagedCache(m, 2, page_size=16)
    cache.release(1)
    before = _state(cache)
    for _ in range(2):
        with pytest.raises(error, match="block size|exceed|HIP devices only"):
            decode.prefill(m, torch.zeros(2, width, dtype=torch.long), cache, counts)
        assert _state(cache) == before


@pytest.mark.parametrize("held", [[5, 9], [16, 31], [16, 0]])
def test_step_that_raises(held):
    """Also where the step had added pages."""
    m = _model()
    cache = decode.PagedCache(m, 2, page_size=16)
    cache.reserve(held)
    if held[1] == 0:
        cache.release(1)
    cache.lengths.copy_(torch.tensor(held))
    before = _state(cache)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="HIP devices only"):
            decode.decode_step(m, torch.tensor([1, 2]), cache)
        assert _state(cache) == before
    cache.reserve([3, 2])                          # and it goes on
    assert cache._held == [held[0] + 3, held[1] + 2 if held[1] else 0]


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["block", "head"])
def test_the_sequences_go_on_after_a_failure(where, monkeypatch):
    """A layer or the output projection that raises once, in the prefill and in
    a step that needs a new page: the same logits as without it."""
    from test_gpu_decode import _plain_model
    m = _plain_model(frozen=(1,))
    x = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(5)).cuda()

    def failing(call):
        layer = m.lm_head if where == "head" else m.transformer.h[1].mlp
        with monkeypatch.context() as p:
            p.setattr(layer, "forward", lambda *a: (_ for _ in ()).throw(MemoryError("no room")))
            with pytest.raises(MemoryError):
                call()

    cache, twin = decode.PagedCache(m, 2, page_size=16), decode.PagedCache(m, 2, page_size=16)
    failing(lambda: decode.prefill(m, x[:, :32], cache, [32, 15]))
    a, b = decode.prefill(m, x[:, :32], cache, [32, 15]), decode.prefill(m, x[:, :32], twin, [32, 15])
    assert torch.equal(a, b)
    for i in range(3):
        failing(lambda: decode.decode_step(m, x[:, 32 + i], cache))
        assert torch.equal(decode.decode_step(m, x[:, 32 + i], cache), decode.decode_step(m, x[:, 32 + i], twin))
        assert cache._held == twin._held and cache.lengths.tolist() == twin.lengths.tolist()
