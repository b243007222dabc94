"""What nanogpt.decode does with prompts, up to the operators (CPU), and their
padding on the device."""
import pytest
import torch

from nanogpt import decode
from test_decode_cache import _model


@pytest.mark.parametrize("pad", [-1, -100, 128])
def test_padding_may_be_any_number(pad, monkeypatch):
    """It is replaced before it reaches the embedding."""
    m = _model()
    x = torch.randint(0, 128, (2, 10), generator=torch.Generator().manual_seed(1))
    x[1, 4:] = pad
    seen = []
    wte = m.transformer.wte.forward
    monkeypatch.setattr(m.transformer.wte, "forward", lambda t: seen.append(t.clone()) or wte(t))
    with pytest.raises(RuntimeError, match="HIP devices only"):   # past the embedding
        decode.prefill(m, x, decode.PagedCache(m, 2, page_size=16), [10, 4])
    assert torch.equal(seen[0][0], x[0]) and torch.equal(seen[0][1, :4], x[1, :4])
    assert bool(((seen[0] >= 0) & (seen[0] < 128)).all())
    assert int(x[1, 9]) == pad                   # the caller's prompts stay as they are


@pytest.mark.gpu
def test_padding_does_not_reach_the_logits():
    from test_model import _small_model
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=torch.bfloat16)
    x = x.repeat(2, 1)[:, :40]
    got = []
    for pad in (7, -1, 50304):
        p = x.clone()
        p[1, 13:] = pad
        cache = decode.PagedCache(m, 2, page_size=16)
        a = decode.prefill(m, p, cache, [40, 13])
        got.append((a, decode.decode_step(m, x[:, 0], cache)))
    assert all(torch.equal(u, v) for g in got[1:] for u, v in zip(g, got[0]))
    tokens, _ = decode.generate(m, p, 5, [40, 13])
    assert torch.equal(tokens, decode.generate(m, x, 5, [40, 13])[0])
