"""nanogpt.train with modules of the caller's own in the model: what they compute is
part of the pass, as in GPT.forward_hidden (CPU: the fused operators in plain torch,
so both paths are the same float32 operations)."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import kernel
from nanogpt import train
from nanogpt.model import GPT, Block
from test_decode_cache import _model as _bare
from test_model_substitutes import _Attention


def _embed(tokens, weight, scale=1.0, ignore_index=-100, dtype=None):
    skip, out = tokens == ignore_index, (tokens < 0) | (tokens >= weight.size(0))
    y = F.embedding(tokens.clamp(0, weight.size(0) - 1), weight) * scale
    return y.masked_fill(out[..., None], float("nan")).masked_fill(skip[..., None], 0.0)


def _norm(x, delta, weight, bias=None, eps=1e-5, dtype=None):
    r = x if delta is None else x + delta
    return r, F.layer_norm(r, weight.shape, weight, bias, eps)


def _mlp(x, w_fc, w_proj, b_fc=None, b_proj=None):
    return F.linear(F.gelu(F.linear(x, w_fc, b_fc)), w_proj, b_proj)


@pytest.fixture(autouse=True)
def calls(monkeypatch):
    """The operators in plain torch; the names of those that ran."""
    made = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)   # asks for a device
    for name, f in (("embed_tokens", _embed), ("add_layernorm", _norm), ("mlp_packed", _mlp)):
        monkeypatch.setattr(kernel, name, lambda *a, _n=name, _f=f, **k: (made.append(_n), _f(*a, **k))[1])
    return made


def _model():
    m = _bare()
    torch.manual_seed(7)
    for blk in m.transformer.h:
        blk.attn = _Attention(blk.attn)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(torch.randn_like(p) * 0.1)
    return m


IDX = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(1))


def _same(m, packed=True):
    """Hidden states and every gradient of both paths."""
    out = []
    for f in (lambda: m.forward_hidden(IDX), lambda: train.forward_hidden(m, IDX, packed)):
        m.zero_grad(set_to_none=True)
        h = f()
        (h * torch.linspace(-1, 1, h.numel()).view_as(h)).sum().backward()
        out.append((h.detach(), {n: p.grad for n, p in m.named_parameters() if p.grad is not None}))
    (a, ga), (b, gb) = out
    assert torch.equal(a, b)
    assert ga.keys() == gb.keys()
    for n in ga:
        # the same terms, added in another order at most
        assert (ga[n] - gb[n]).norm() <= 1e-5 * ga[n].norm(), n
    return ga


class _Adapter(nn.Linear):
    """A linear layer with a low-rank addition."""

    def __init__(self, inner, rank=3):
        super().__init__(inner.in_features, inner.out_features, inner.bias is not None)
        self.weight, self.bias = inner.weight, inner.bias
        self.down = nn.Parameter(torch.randn(rank, inner.in_features) * 0.1)
        self.up = nn.Parameter(torch.randn(inner.out_features, rank) * 0.1)

    def forward(self, x):
        return super().forward(x) + x @ self.down.t() @ self.up.t()


def _hook(module, args, out):
    return out * 1.5


def _pre_hook(module, args):
    return (args[0] * 0.5,)


def test_plain_model_is_fused(calls):
    m = _model()
    _same(m)
    assert calls == ["embed_tokens"] + ["add_layernorm", "add_layernorm", "mlp_packed"] * 2 + ["add_layernorm"]


# ---- inside the MLP ---------------------------------------------------------------

@pytest.mark.parametrize("act", [nn.SiLU(), nn.ReLU(), nn.Identity(), nn.GELU(approximate="tanh")], ids=lambda a: str(a))
def test_activations(act, calls):
    m = _model()
    m.transformer.h[0].mlp.gelu = act
    _same(m)
    assert calls.count("mlp_packed") == 1


@pytest.mark.parametrize("name", ["c_fc", "c_proj"])
def test_adapted_projections(name, calls):
    m = _model()
    mlp = m.transformer.h[1].mlp
    setattr(mlp, name, _Adapter(getattr(mlp, name)))
    grads = _same(m)
    assert {f"transformer.h.1.mlp.{name}.{p}" for p in ("weight", "down", "up")} <= grads.keys()
    assert calls.count("mlp_packed") == 1


@pytest.mark.parametrize("name", ["", "c_fc", "gelu", "c_proj"])
def test_hooked_mlps(name, calls):
    for add in (lambda t: t.register_forward_hook(_hook), lambda t: t.register_forward_pre_hook(_pre_hook),
                lambda t: t.register_full_backward_hook(lambda *a: (a[1][0] * 2,))):
        m = _model()
        add(m.transformer.h[1].mlp.get_submodule(name))
        _same(m)
    m = _model()
    target = m.transformer.h[1].mlp.get_submodule(name)
    own = target.forward
    target.forward = lambda x: own(x) * 0.25
    _same(m)
    assert calls.count("mlp_packed") == 4


# ---- the norms --------------------------------------------------------------------

class _RMSNorm(nn.Module):
    def __init__(self, n):
        super().__init__()
        self.gain = nn.Parameter(torch.linspace(0.5, 1.5, n))

    def forward(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-3) * self.gain


def _owner(m, name):
    return m.transformer if name == "ln_f" else m.transformer.h[1]


@pytest.mark.parametrize("name", ["ln_1", "ln_2", "ln_f"])
@pytest.mark.parametrize("other", [lambda: nn.LayerNorm(128, eps=0.5), lambda: _RMSNorm(128),
                                   lambda: nn.LayerNorm(128, elementwise_affine=False), nn.Identity],
                         ids=["eps", "rms", "bare", "none"])
def test_other_norms(name, other, calls):
    m = _model()
    _owner(m, name).add_module(name, other())
    _same(m)
    assert calls.count("add_layernorm") == 4


@pytest.mark.parametrize("name", ["ln_1", "ln_2", "ln_f"])
def test_hooked_norms(name, calls):
    for add in (lambda t: t.register_forward_hook(_hook), lambda t: t.register_forward_pre_hook(_pre_hook),
                lambda t: t.register_full_backward_hook(lambda *a: (a[1][0] * 2,))):
        m = _model()
        add(getattr(_owner(m, name), name))
        _same(m)
    assert calls.count("add_layernorm") == 12


# ---- blocks -----------------------------------------------------------------------

class _Scaled(Block):
    def forward(self, x, rope=None, **sink):
        return x + 0.5 * (super().forward(x, rope=rope, **sink) - x)


class _Wrapper(nn.Module):
    """A block without the names of Block's parts."""

    def __init__(self, inner):
        super().__init__()
        self.inner, self.gain = inner, nn.Parameter(torch.tensor(0.7))

    def forward(self, x, rope=None):
        return self.inner(x, rope=rope) * self.gain


@pytest.mark.parametrize("at", [(0,), (1,), (0, 1)])
def test_other_blocks(at, calls):
    def scaled(m, i):
        m.transformer.h[i].__class__ = _Scaled

    def wrapped(m, i):
        m.transformer.h[i] = _Wrapper(m.transformer.h[i])

    def hooked(m, i):
        m.transformer.h[i].register_forward_hook(_hook)

    def own_forward(m, i):
        blk = m.transformer.h[i]
        was = blk.forward
        blk.forward = lambda x, **k: was(x, **k) * 2

    for change in (scaled, wrapped, hooked, own_forward):
        m = _model()
        for i in at:
            change(m, i)
        grads = _same(m)
        assert change is not wrapped or {f"transformer.h.{i}.gain" for i in at} <= grads.keys()
    assert calls.count("mlp_packed") == 4 * (2 - len(at))


def test_no_blocks():
    m = _model()
    m.transformer.h = nn.ModuleList()
    _same(m)


# ---- the embedding ----------------------------------------------------------------

class _Embedding(nn.Embedding):
    def forward(self, idx):
        return super().forward(idx) * 1.5


def test_other_embeddings(calls):
    def subclass(m):
        m.transformer.wte.__class__ = _Embedding

    def replaced(m):
        m.transformer.wte = nn.Sequential(nn.Embedding(128, 16), nn.Linear(16, 128))

    def padded(m):
        m.transformer.wte.padding_idx = int(IDX[0, 3])       # a row without gradient

    def by_frequency(m):
        m.transformer.wte.scale_grad_by_freq = True

    def hooked(m):
        m.transformer.wte.register_forward_hook(_hook)

    for change in (subclass, replaced, padded, by_frequency, hooked):
        m = _model()
        # beside the head's weight, whose gradient would be the sum of both
        m.transformer.wte.weight = nn.Parameter(m.transformer.wte.weight.detach().clone())
        change(m)
        grads = _same(m)
        if change is padded:
            assert not grads["transformer.wte.weight"][int(IDX[0, 3])].any()
    assert "embed_tokens" not in calls


def test_renormalised_embedding(calls):
    """max_norm changes the weight in place; without a gradient, as nn.Embedding asks."""
    m = _model()
    m.transformer.wte.max_norm = 0.25
    m.transformer.wte.weight.requires_grad_(False)
    _same(m)
    assert m.transformer.wte.weight[IDX[0, 0]].norm() <= 0.2501 and "embed_tokens" not in calls


def test_sparse_embedding(calls):
    m = _model()
    m.transformer.wte.weight = nn.Parameter(m.transformer.wte.weight.detach().clone())
    m.transformer.wte.sparse = True
    train.forward_hidden(m, IDX).sum().backward()
    assert m.transformer.wte.weight.grad.is_sparse and "embed_tokens" not in calls


# ---- the model --------------------------------------------------------------------

class _Inputs(GPT):
    def prepare_inputs(self, idx):
        x, rope = super().prepare_inputs(idx)
        return x * 2, rope


class _Hidden(GPT):
    def forward_hidden(self, idx, sinks=None):
        return super().forward_hidden(idx, sinks) * 2


class _Logits(GPT):
    def forward_all_positions(self, idx):
        return super().forward_all_positions(idx) * 2


def test_inputs_of_the_model(calls):
    m = _model()
    m.__class__ = _Inputs
    _same(m)
    assert "embed_tokens" not in calls


class _Fused(GPT):
    """The pass as the model's own hidden states."""

    def forward_hidden(self, idx, sinks=None):
        return train.forward_hidden(self, idx)


@pytest.mark.parametrize("kind", [GPT, _Inputs, _Logits, _Hidden, _Fused])
def test_logits_of_the_model(kind, monkeypatch):
    monkeypatch.setattr(kernel, "token_logprobs", lambda logits, tokens, **kw: logits)
    m = _model()
    m.__class__ = kind
    assert torch.equal(train.token_logprobs(m, IDX, IDX), m.token_logprobs(IDX, IDX))


# ---- tokens -----------------------------------------------------------------------

@pytest.mark.parametrize("bad", [-100, -1, 128, 1 - 2 ** 63, 2 ** 63 - 1])
def test_tokens_outside_the_vocabulary(bad):
    """No row of zeros for any of them: the sequence is NaN and the others as they are."""
    m = _model()
    idx = IDX.clone()
    idx[1, 4] = bad
    h, want = train.forward_hidden(m, idx), train.forward_hidden(m, IDX)
    assert h[1, 4].isnan().all() and torch.equal(h[0], want[0])


# ---- branches that do not meet the residual ------------------------------------------

class _Branch(nn.Module):
    """An MLP whose result has a dtype or a shape of its own."""

    def __init__(self, dtype=None, lead=None):
        super().__init__()
        self.dtype, self.lead, self.gain = dtype, lead, nn.Parameter(torch.tensor(0.3))

    def forward(self, x):
        y = (x if self.lead is None else x.mean(dim=(0, 1)).view(*self.lead, -1)) * self.gain
        return y if self.dtype is None else y.to(self.dtype)


@pytest.mark.parametrize("lead", [(), (1,), (1, 1)])
@pytest.mark.parametrize("at", [0, 1])
def test_broadcast_branches(lead, at, monkeypatch):
    """Added as torch adds them, ahead of a norm that takes one shape only."""
    def strict(x, delta, *a, **k):
        assert delta is None or delta.shape == x.shape
        return _norm(x, delta, *a, **k)

    monkeypatch.setattr(kernel, "add_layernorm", strict)
    m = _model()
    m.transformer.h[at].mlp = _Branch(lead=lead)
    assert f"transformer.h.{at}.mlp.gain" in _same(m)
