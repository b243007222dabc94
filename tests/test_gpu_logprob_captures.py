"""Captures of token_logprobs' gradient that torch's engine would not survive
are refused before anything is recorded, however the logits come from their
leaf."""
import pytest
import torch

import kernel

pytestmark = pytest.mark.gpu

CHAINS = dict(slice_of_rows=lambda x: x[..., :900].unflatten(0, (2, 2)), cast=lambda x: x.double().float(),
              transposed=lambda x: x.t().contiguous().t(), row=lambda x: x[2][5:], shifted=lambda x: x[:-1, 3:].unsqueeze(0) * 0.5)


@pytest.mark.parametrize("chain", sorted(CHAINS))
def test_logits_derived_from_a_leaf(chain):
    x = torch.randn(4, 1000, device="cuda", requires_grad=True)
    make = CHAINS[chain]
    t = torch.zeros(make(x).shape[:-1], dtype=torch.long, device="cuda")
    alive = kernel.token_logprobs(make(x), t)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kernel.token_logprobs(make(x), t)
    torch.cuda.synchronize()
    assert torch.isfinite(alive.logp).all()


@pytest.mark.parametrize("chain", sorted(CHAINS))
def test_captured_gradients_of_derived_logits(chain):
    """With no eager graph of the leaf: captured, replayed, and right."""
    x = torch.randn(4, 1000, device="cuda", requires_grad=True)
    y = x.detach().clone().requires_grad_()
    make = CHAINS[chain]
    t = torch.zeros(make(x).shape[:-1], dtype=torch.long, device="cuda")
    (want,) = torch.autograd.grad(kernel.token_logprobs(make(y), t).logp.sum(), y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(kernel.token_logprobs(make(x), t).logp.sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(kernel.token_logprobs(make(x), t).logp.sum(), x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
