"""nanogpt.train with modules of the caller's own in the model against the model's own
path, on the kernels: float32, the bounds of test_gpu_train_model.test_float32."""
import copy

import pytest
import torch
import torch.nn as nn

from nanogpt import train
from test_gpu_train_model import _batch, _loss_and_grads, _model, _near
from test_train_substitutes import _Adapter, _Branch, _hook, _Scaled, _Wrapper
from train_cases import DEV

pytestmark = pytest.mark.gpu


def _same(m, packed):
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt, packed=packed).logp)
    assert (a - b).abs().max() <= 6e-4
    _near(gb, ga, 0.1 if packed else 6e-4)
    return ga


@pytest.mark.parametrize("packed", [False, True])
def test_mlps(packed):
    """One of the two layers stays packed where packed is asked for."""
    m = _model()
    m.transformer.h[0].mlp.gelu = nn.SiLU()
    _same(m, packed)
    m = _model()
    mlp = m.transformer.h[1].mlp
    mlp.c_fc, mlp.c_proj = _Adapter(mlp.c_fc).to(DEV), _Adapter(mlp.c_proj).to(DEV)
    grads = _same(m, packed)
    assert sum("down" in n or "up" in n for n in grads) == 4
    m = _model()
    m.transformer.h[0].mlp.c_fc.register_forward_hook(_hook)
    _same(m, packed)


@pytest.mark.parametrize("packed", [False, True])
def test_norms(packed):
    m = _model()
    m.transformer.h[0].ln_1 = nn.LayerNorm(128, eps=0.5).to(DEV)
    m.transformer.h[1].ln_2 = nn.LayerNorm(128, eps=0.5).to(DEV)
    _same(m, packed)
    m = _model()
    m.transformer.ln_f = nn.LayerNorm(128, eps=0.5).to(DEV)
    m.transformer.h[0].ln_2.register_forward_hook(_hook)
    _same(m, packed)


def test_norms_under_autocast():
    """float32 norms of the caller's own between bf16 branches (the bound of
    test_gpu_train_model.test_autocast)."""
    m = _model(frozen=False)
    m.transformer.h[1].ln_1 = nn.LayerNorm(128, eps=0.5).to(DEV)
    m.transformer.ln_f = nn.LayerNorm(128, eps=0.5).to(DEV)
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    with torch.autocast("cuda", torch.bfloat16):
        _, own = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
        b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt, packed=False).logp)
    assert (a - b).abs().max() <= 10 * 2.0 ** -8 * 4
    _near(gb, ga, 10 * 2.0 ** -8, own)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind", [_Scaled, _Wrapper])
def test_blocks(kind, packed):
    """A block of the caller's own before and behind one that is fused."""
    for at in (0, 1):
        m = _model()
        blocks = m.transformer.h
        if kind is _Scaled:
            blocks[at].__class__ = _Scaled
        else:
            blocks[at] = _Wrapper(blocks[at]).to(DEV)
        _same(m, packed)


def test_embeddings():
    m = _model()
    m.transformer.wte = nn.Sequential(nn.Embedding(211, 16), nn.Linear(16, 128)).to(DEV)
    _same(m, True)
    m = _model()
    m.transformer.wte.weight = nn.Parameter(m.transformer.wte.weight.detach().clone())
    m.transformer.wte.padding_idx = 5
    idx, _ = _batch(m)
    assert (idx == 5).any()
    grads = _same(m, True)
    assert not grads["transformer.wte.weight"][5].any()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("bad", [-100, 211])
def test_tokens_outside_the_vocabulary(bad, dtype):
    """What such a token reaches is NaN, and the loss with it; the other sequences are
    as they were."""
    m = _model(frozen=False)
    idx, nxt = _batch(m)
    want = train.token_logprobs(m, idx, nxt).logp.detach()
    idx[1, 60] = bad
    got = train.token_logprobs(m, idx.to(dtype), nxt).logp.detach()
    assert got[1, 60:].isnan().all()
    assert torch.equal(got[::2], want[::2])


@pytest.mark.parametrize("lead", [None, (1,), (1, 1)])
def test_branches_of_another_type_or_shape(lead):
    """A float32 branch widens a bf16 residual, as torch's sum does (the model's norms
    take it under autocast).  Against the same weights in float32, with the bounds of
    test_gpu_train_model.test_bf16_model (this residual has more bits) and, for q and k,
    what the model's own path shows of the cancellation in their gradients."""
    m = _model(dtype=torch.bfloat16, frozen=False)
    m.transformer.h[0].mlp = _Branch(torch.float32, lead).to(DEV)
    idx, nxt = _batch(m)
    whole = copy.deepcopy(m).float()
    a, ga = _loss_and_grads(whole, lambda: whole.token_logprobs(idx, nxt).logp)
    with torch.autocast("cuda", torch.bfloat16):
        _, own = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
        b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp)
    assert (a - b).abs().max() <= 20 * 2.0 ** -8 * 4
    _near(gb, ga, 20 * 2.0 ** -8 + 0.1, own)
