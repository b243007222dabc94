"""What a captured decoding step reads stays where it is (CPU): the step's row
normalisers of trainable patterns, and the packed projection weights."""
import pytest
import torch

from nanogpt import decode
from test_trainable_patterns import _model, restore_dispatch  # noqa: F401


@pytest.fixture
def patterns(monkeypatch, restore_dispatch):  # noqa: F811
    """A model with trainable patterns whose normalisers run on the CPU."""
    import supplement
    from kernel import decomposed_logz
    from supplement import trainable_patterns as module
    calls = []

    def normalisers(alpha, rho, length):
        calls.append(length)
        z = torch.zeros(alpha.shape)
        z[:, :length] = decomposed_logz(alpha.detach()[:, :length], rho.detach()[:, :length])
        return z

    monkeypatch.setattr(module, "normalisers", normalisers)
    m = _model()
    supplement.enable(m)
    return m, m.transformer.h[0].attn, m._saf_patterns, calls


def _want(attn):
    from kernel import decomposed_logz
    return decomposed_logz(attn.dyn_alpha.detach(), attn.dyn_rho.detach())


def test_step_normalisers_outlive_prefills(patterns):
    m, attn, owner, calls = patterns
    z = owner.step_inputs(attn)["z"]
    assert torch.equal(z, _want(attn))
    for T in (16, 48, 64):
        owner.kernel_inputs(attn, T)
    n = len(calls)
    assert owner.step_inputs(attn)["z"] is z and len(calls) == n    # neither replaced nor computed again


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_changed_patterns_refresh_the_step_normalisers_in_place(patterns, mode):
    m, attn, owner, calls = patterns
    with mode():
        z = owner.step_z(attn)
    with torch.no_grad():
        attn.dyn_alpha[1, :10] += 0.5
    with mode():
        assert owner.step_z(attn) is z
    assert torch.equal(z, _want(attn))
    attn.dyn_rho.data[1, 3] -= 1.0          # no version counter moves
    owner.invalidate()
    assert owner.step_z(attn) is z and torch.equal(z, _want(attn))


def test_cache_check_makes_them_before_a_capture(patterns):
    m, attn, owner, calls = patterns
    cache = decode.PagedCache(m, 1, page_size=16)
    cache.check(m)
    assert calls == [64] and owner.step_z(attn) is owner.step_inputs(attn)["z"] and calls == [64]


@pytest.mark.parametrize("what", ["z_for", "step_z"])
def test_a_capture_keeps_nothing(patterns, what, monkeypatch):
    from supplement import trainable_patterns as module
    m, attn, owner, calls = patterns
    call = (lambda: owner.z_for(attn, 64)) if what == "z_for" else (lambda: owner.step_z(attn))
    monkeypatch.setattr(module, "_capturing", lambda t: True)
    recorded = call()
    monkeypatch.setattr(module, "_capturing", lambda t: False)
    z = call()
    assert z is not recorded and torch.equal(z, _want(attn))
    monkeypatch.setattr(module, "_capturing", lambda t: True)
    if what == "z_for":
        assert call() is not z              # a replay follows the parameters
    else:
        assert call() is z                  # refreshed in place, outside the capture


def test_packed_weights_are_refreshed_in_place():
    """eval() again, or changed weights: the same storage with the current
    rows, whichever mode made it; other live heads: their rows."""
    m = _model().eval()
    attn = m.transformer.h[1].attn
    attn._refresh_freeze_cache()
    with torch.inference_mode():
        w, b = attn._infer_weight_cache()
    assert b is None and torch.equal(w[:128], attn.q_proj.weight)
    m.train()
    m.eval()
    with torch.no_grad():
        attn.q_proj.weight[5] += 1.0
        assert attn._infer_weight_cache()[0] is w and torch.equal(w[:128], attn.q_proj.weight)
    attn.dyn_frozen[0] = True
    attn._refresh_freeze_cache()
    with torch.inference_mode():
        fewer, _ = attn._infer_weight_cache()
    assert torch.equal(fewer[:96], attn.q_proj.weight[32:]) and torch.equal(fewer[192:320], attn.v_proj.weight)
    m.to(torch.bfloat16)
    with torch.no_grad():
        assert torch.equal(attn._infer_weight_cache()[0][:96], attn.q_proj.weight[32:])


def test_packed_biases_are_refreshed_in_place():
    from nanogpt.model import GPT, GPTConfig
    torch.manual_seed(0)
    m = GPT(GPTConfig(block_size=64, vocab_size=256, n_layer=1, n_head=4, n_embd=128, bias=True,
                      rand_attn_prior_repr="dense")).eval()
    attn = m.transformer.h[0].attn
    attn._refresh_freeze_cache()
    with torch.no_grad():
        b = attn._infer_weight_cache()[1]
        attn.v_proj.bias += 2.0
        attn.v_proj.weight += 1.0
        assert attn._infer_weight_cache()[1] is b and torch.equal(b[256:384], attn.v_proj.bias)


@pytest.mark.parametrize("name", ["q_proj", "k_proj", "v_proj"])
def test_a_changed_bias_alone_is_noticed(name):
    from nanogpt.model import GPT, GPTConfig
    torch.manual_seed(0)
    m = GPT(GPTConfig(block_size=64, vocab_size=256, n_layer=1, n_head=4, n_embd=128, bias=True,
                      rand_attn_prior_repr="dense")).eval()
    attn = m.transformer.h[0].attn
    attn._refresh_freeze_cache()
    with torch.no_grad():
        b = attn._infer_weight_cache()[1]
        getattr(attn, name).bias.add_(2.0)
        at = 128 * ["q_proj", "k_proj", "v_proj"].index(name)
        assert torch.equal(attn._infer_weight_cache()[1][at:at + 128], getattr(attn, name).bias)
        assert attn._infer_weight_cache()[1] is b
        vb, qkb = attn._split_weight_cache()[1], attn._split_weight_cache()[3]
        getattr(attn, name).bias.mul_(-1.0)
        got = torch.cat([attn._split_weight_cache()[3], attn._split_weight_cache()[1]])
        assert torch.equal(got[at:at + 128], getattr(attn, name).bias) and got.numel() == vb.numel() + qkb.numel()
