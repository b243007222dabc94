"""What a captured decoding step reads stays where it is (CPU): the step's row
normalisers of trainable patterns."""
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
