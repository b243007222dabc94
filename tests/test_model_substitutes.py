"""Blocks and attention modules of the caller's own, called as before the
cache's sinks were there (CPU)."""
import torch
import torch.nn as nn

from test_decode_cache import _model


class _Attention(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, rope=None):
        assert rope is not None
        return self.inner.c_proj(x)


class _Block(nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, rope=None):
        return self.inner(x, rope=rope)


def test_forward_through_substitutes():
    m = _model()
    for blk in m.transformer.h:
        blk.attn = _Attention(blk.attn)
    x = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(1))
    want = m.forward_all_positions(x)
    assert torch.isfinite(want).all()
    for i, blk in enumerate(m.transformer.h):
        m.transformer.h[i] = _Block(blk)
    assert torch.equal(m.forward_all_positions(x), want)
