"""Host side of nanogpt.decode: what the cache refuses, and what a refusal
leaves as it was (CPU)."""
import pytest
import torch

from nanogpt import decode
from nanogpt.model import GPT, GPTConfig


def _model(T=64):
    torch.manual_seed(3)
    cfg = GPTConfig(block_size=T, vocab_size=128, n_layer=2, n_head=4, n_embd=128, bias=False,
                    position_encoding="rope", rand_attn_prior_repr="dense")
    return GPT(cfg).eval()


def test_changed_live_heads_are_seen_after_another_forward():
    """A forward between the change and the step refreshes the model's freeze
    tables; the cache still belongs to the old live heads."""
    m = _model()
    for blk in m.transformer.h:
        blk.attn.freeze_heads([1], torch.rand(1, 64, 64))
    cache = decode.PagedCache(m, 1, page_size=16)
    cache.check(m)
    for attn in m.attn_modules():
        attn._fz_dirty = True              # refreshed with the same heads: still good
        attn._refresh_freeze_cache()
    cache.check(m)
    attn = m.attn_modules()[1]
    attn.dyn_frozen[1], attn.dyn_frozen[2] = False, True   # as many live heads, but others
    attn._fz_dirty = True
    attn._refresh_freeze_cache()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="live heads changed"):
            cache.check(m)


def test_refused_prefill_changes_nothing():
    m = _model()
    cache = decode.PagedCache(m, 2, page_size=16, n_pages=3)
    cache.release(1)
    with pytest.raises(ValueError, match="used up"):
        decode.prefill(m, torch.zeros(2, 40, dtype=torch.long), cache)
    assert cache._on == [True, False] and cache.active.tolist() == [1, 0]
    assert cache._held == [0, 0] and len(cache._free) == 3
    assert (cache.page_table == -1).all()


@pytest.mark.parametrize("token", [-1, -100, 128])
def test_inactive_sequences_ignore_their_token(token, monkeypatch):
    """Also one that is no token at all, before it reaches the embedding."""
    m = _model()
    cache = decode.PagedCache(m, 2, page_size=16)
    cache.release(1)
    seen = []
    wte = m.transformer.wte.forward
    monkeypatch.setattr(m.transformer.wte, "forward", lambda t: seen.append(t.clone()) or wte(t))
    with pytest.raises(RuntimeError, match="HIP devices only"):   # past the embedding
        decode.decode_step(m, torch.tensor([5, token]), cache)
    assert seen[0].reshape(-1)[0] == 5 and 0 <= int(seen[0].reshape(-1)[1]) < 128
