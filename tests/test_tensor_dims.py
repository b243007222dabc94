"""Tensors of more dimensions than a descriptor of the C-ABI has (4): refused before
one is written, which would write behind it."""
import pytest
import torch

import kernel
from kernel import _ext

DIMS = [0, 2, 4, 5, 6, 12, 40]


@pytest.mark.parametrize("n", DIMS)
def test_norm_vectors(n):
    """Weights and biases are vectors, whatever the device."""
    x, w = torch.zeros(2, 8), torch.zeros(8)
    bad = torch.zeros([1] * max(n - 1, 0) + [8] * min(n, 1))
    with pytest.raises(ValueError, match="weight must be"):
        kernel.add_layernorm(x, None, bad)
    with pytest.raises(ValueError, match="bias must be"):
        kernel.add_layernorm(x, None, w, bad)
    with pytest.raises(ValueError, match="x must have channels"):
        kernel.add_layernorm(x[0, 0], None, w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 6, 12])
def test_descriptors(n):
    """The binding's own entry points, without the shapes that kernel.* gives them."""
    x = torch.zeros([1] * (n - 1) + [8], device="cuda")
    t = torch.zeros(1, dtype=torch.long, device="cuda")
    b = _ext.bind()
    with pytest.raises(ValueError, match="at most 4 dimensions"):
        b.token_logprobs(x, t, 0, False, 1.0, -100)
    with pytest.raises(ValueError, match="at most 4 dimensions"):
        b.token_logprobs(x.view(1, 8), t.view([1] * n), 0, False, 1.0, -100)
    with pytest.raises(ValueError, match="weight must be"):
        kernel.add_layernorm(x.view(1, 8), None, x)
    # operands of rows take any number of dimensions
    w = torch.ones(8, device="cuda")
    assert kernel.add_layernorm(x, x, w)[1].shape == x.shape
    assert kernel.gelu_packed(x).shape == x.shape
    assert kernel.embed_tokens(t.view([1] * n), x.view(1, 8)).shape == (*[1] * n, 8)
