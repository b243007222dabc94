"""nanogpt.train against the model's own path: the same loss, the same gradients,
up to the rounding of the two paths and of the 8-bit activations."""
import pytest
import torch

import kernel
from nanogpt import train
from nanogpt.model import GPT, GPTConfig
from train_cases import BF16, DEV, F32, in_use

pytestmark = pytest.mark.gpu


def _model(dtype=F32, bias=True, pos="rope", layers=2, frozen=True, V=211, T=128, seed=3):
    torch.manual_seed(seed)
    m = GPT(GPTConfig(block_size=T, vocab_size=V, n_layer=layers, n_head=4, n_embd=128, bias=bias, position_encoding=pos)).to(DEV)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() == 1:
                p.add_(torch.randn_like(p) * 0.1)
    if frozen:
        d = torch.arange(T, dtype=F32, device=DEV)
        for l, b in enumerate(m.transformer.h):
            b.attn.freeze_heads_decomposed([l % 4], torch.zeros(1, T, device=DEV), (-0.02 * (l + 1) * d)[None])
            b.attn.freeze_heads([(l + 2) % 4], torch.rand(1, T, T, device=DEV))
    return m.to(dtype)


def _batch(m, B=3, T=100, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(0, m.config.vocab_size, (B, T), device=DEV, generator=g) for _ in range(2)]


def _loss_and_grads(m, f):
    m.zero_grad(set_to_none=True)
    logp = f()
    (-logp.mean()).backward()
    return logp.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}


def _near(a, b, rel, own=None):
    """Norms of a - b within rel of b's.  own: the model's own path in a's types.  The
    gradients of q and k come from P (dP - delta), where dP and delta, each rounded to
    bf16 inside the attention, cancel for the nearly even P of a new model: with |dP| =
    c |dP - delta| their relative error is c times a rounding's, c unknown here.  The
    model's own path runs the same attention and shows that error itself; two such
    errors of one cause differ by their sum at most, twice it with equal sizes."""
    assert a.keys() == b.keys()
    for n in a:
        err, size = (a[n].double() - b[n].double()).norm(), b[n].double().norm()
        if n.endswith("k_proj.bias"):
            # one vector c on every key adds q . c to all scores of a row, which the
            # softmax does not see: without rotation this gradient is zero, a sum of
            # terms that cancel, each off relatively to itself.  The queries' bias has
            # terms of the same size that do not cancel
            size = max(size, b[n.replace("k_proj", "q_proj")].double().norm())
        cause = 2 * (own[n].double() - b[n].double()).norm() if own and ("q_proj" in n or "k_proj" in n) else 0
        assert err <= rel * size + cause + 1e-12, (n, float(err / size))


@pytest.mark.parametrize("pos", ["rope", "learned_absolute"])
@pytest.mark.parametrize("bias", [True, False])
def test_float32(pos, bias):
    """Whole activations: two float32 evaluations of one function.  A path of 2
    layers is about 10 products of up to 512 terms deep, each off by K U of its
    magnitudes relatively at most, sqrt(K) U in the norm over many elements, and as
    many norms: 10 x 2 x 512 U = 6e-4 bounds the gradients' norms."""
    m = _model(bias=bias, pos=pos)
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt, packed=False).logp)
    assert (a - b).abs().max() <= 6e-4
    _near(gb, ga, 6e-4)
    # packed: the forward pass is the same to the bit of its GELU (16 U relative)
    c, gc = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp)
    assert (a - c).abs().max() <= 6e-4
    # the held values are off by a 128th of their block's largest at most, uniformly
    # inside a step: for the weights' products that is the relative error of x (its
    # block's largest is up to 4 deviations: 4 / 64 / sqrt(12) = 0.018), for the
    # GELU's slope at most 0.8 of the step's error of arguments around 1 beside a
    # slope of 0.5 rms: 0.8 x 0.018 / 0.5 = 0.03; two layers of both
    _near(gc, ga, 0.1)


def test_autocast():
    """float32 weights and residual stream, bf16 branches: 2^-8 a rounding, about ten
    along the path of 2 layers."""
    m = _model(frozen=False)
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    with torch.autocast("cuda", BF16):
        _, own = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    for packed in (False, True):
        with torch.autocast("cuda", BF16):
            h = train.forward_hidden(m, idx, packed)
            assert h.dtype == BF16
        del h
        with torch.autocast("cuda", BF16):
            b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt, packed=packed).logp)
        assert all(g.dtype == F32 for g in gb.values())
        assert (a - b).abs().max() <= 10 * 2.0 ** -8 * 4          # logits of magnitude up to 4
        _near(gb, ga, 10 * 2.0 ** -8 + (0.1 if packed else 0), own)


def test_bf16_model():
    m = _model(dtype=BF16)
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp)
    assert (a - b).abs().max() <= 20 * 2.0 ** -8 * 4              # both paths round
    _near(gb, ga, 20 * 2.0 ** -8 + 0.1)


def test_same_bits_every_time():
    """Two passes over one batch: the framework's operators add in a fixed order."""
    m = _model(dtype=BF16, frozen=False)
    idx, nxt = _batch(m)
    runs = [_loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp) for _ in range(2)]
    assert torch.equal(runs[0][0], runs[1][0])
    for n in ("transformer.ln_f.weight", "transformer.ln_f.bias"):
        assert torch.equal(runs[0][1][n], runs[1][1][n])


def test_trainable_patterns():
    """alpha and rho of a layer that trains them: the same gradients on both paths (the
    bound of test_bf16_model)."""
    import supplement
    m = _model(dtype=BF16, bias=False)
    supplement.enable(m)
    idx, nxt = _batch(m)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp)
    assert sum("alpha" in n or "rho" in n for n in gb) == 4
    assert (a - b).abs().max() <= 20 * 2.0 ** -8 * 4
    _near(gb, ga, 20 * 2.0 ** -8 + 0.1)


def test_modules_of_the_callers_own(monkeypatch):
    """Another MLP, or another activation, runs as it is."""
    m = _model()
    idx, nxt = _batch(m)
    m.transformer.h[0].mlp.gelu = torch.nn.GELU(approximate="tanh")
    m.transformer.h[1].mlp = torch.nn.Linear(128, 128).to(DEV)
    monkeypatch.setattr(kernel, "mlp_packed", None)
    a, ga = _loss_and_grads(m, lambda: m.token_logprobs(idx, nxt).logp)
    b, gb = _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt).logp)
    assert (a - b).abs().max() <= 6e-4
    _near(gb, ga, 6e-4)


def test_refusals():
    m = _model(frozen=False)
    with pytest.raises(ValueError, match="block size"):
        train.forward_hidden(m, torch.zeros(1, 129, dtype=torch.long, device=DEV))


def test_capture_is_refused_while_an_eager_graph_lives():
    """Also where only weights of torch's own operators are trained."""
    m = _model(dtype=BF16, frozen=False)
    m.requires_grad_(False)
    for b in m.transformer.h:
        b.attn.q_proj.requires_grad_()
        b.attn.k_proj.requires_grad_()
    idx, nxt = _batch(m)
    alive = train.token_logprobs(m, idx, nxt).logp
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            train.token_logprobs(m, idx, nxt)
    torch.cuda.synchronize()
    assert torch.isfinite(alive).all()


def test_memory():
    """The packed step keeps less: the MLPs' activations in 8 bits."""
    m = _model(dtype=BF16, layers=4, frozen=False)
    idx, nxt = _batch(m, B=32, T=128)
    held = {}
    for packed in (False, True):
        _loss_and_grads(m, lambda: train.token_logprobs(m, idx, nxt, packed=packed).logp)   # workspaces
        torch.cuda.synchronize()
        before = in_use()
        h = train.forward_hidden(m, idx, packed)
        held[packed] = in_use() - before
        del h
    rows, C = 32 * 128, 128
    # 4 layers x (8 + 8 C) bytes of u and gelu(u) against 4 (1 + 1/32) C; x is kept by no
    # other part of the graph, the norm's result being the attention's only in the block before
    saved = 4 * rows * C * (16 - 4 * 33 / 32)
    assert held[False] - held[True] >= saved * 0.95
