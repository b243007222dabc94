"""The decoding operators together, as the GPT uses them: prefill into a paged
cache, one token per sequence and step, greedy generation, graph replays, and
the training loss."""
import pytest
import torch

import kernel
from nanogpt import decode
from nanogpt import model as model_mod
from nanogpt.model import GPT, GPTConfig
from test_model import _cos, _small_model

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _rel(a, b):
    """Relative error of a against b (Frobenius)."""
    return float((a.double() - b.double()).norm() / b.double().norm())


def _plain_model(position_encoding="rope", bias=True, dtype=BF16, frozen=(), T=128, hd=64):
    torch.manual_seed(5)
    cfg = GPTConfig(block_size=T, vocab_size=512, n_layer=2, n_head=4, n_embd=4 * hd, bias=bias,
                    position_encoding=position_encoding, rand_attn_prior_repr="dense")
    m = GPT(cfg).to("cuda", dtype).eval()
    for blk in m.transformer.h:
        if frozen:
            blk.attn.freeze_heads(list(frozen), torch.rand(len(frozen), T, T, device="cuda"))
    return m


def _steps_against_prefill(m, x, start, tol, counts=None):
    """Decode x[:, start:] token by token and compare every step's logits with
    the whole-sequence forward at the same position."""
    B, T = x.shape
    with torch.inference_mode():
        want = m.forward_all_positions(x).float()
    cache = decode.PagedCache(m, B, page_size=16)
    counts = [start] * B if counts is None else counts
    width = max(counts)
    prompt = x[:, :width].clone()
    for b, c in enumerate(counts):
        prompt[b, c:] = 7                      # padding, never to be seen
    logits = decode.prefill(m, prompt, cache, counts)
    at = list(counts)
    for _ in range(T - max(counts)):
        for b in range(B):
            assert _rel(logits[b], want[b, at[b] - 1]) <= tol, (b, at[b])
        tok = torch.stack([x[b, at[b]] for b in range(B)])
        logits = decode.decode_step(m, tok, cache)
        at = [n + 1 for n in at]
    for b in range(B):
        assert _rel(logits[b], want[b, at[b] - 1]) <= tol


# bf16: both sides round activations to 8 bits at every layer, in different
# orders (a few 2^-8 of the logits' norm); float32: a few hundred roundings
@pytest.mark.parametrize("dtype,tol", [(BF16, 3e-2), (FP32, 2e-5)])
def test_steps_match_the_prefill(dtype, tol):
    """Live, dense, decomposed and closed-form heads in every layer."""
    m, x = _small_model(T=192, layers=3, device="cuda", dtype=dtype)
    _steps_against_prefill(m, x, 150, tol)


def test_ragged_batch():
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    x = torch.randint(0, 50257, (3, 128), generator=torch.Generator().manual_seed(2)).cuda()
    _steps_against_prefill(m, x, 0, 3e-2, counts=[100, 1, 33])


@pytest.mark.parametrize("pos", ["rope", "learned_absolute"])
@pytest.mark.parametrize("frozen", [(), (1,), (0, 1, 2, 3)])
@pytest.mark.parametrize("bias", [True, False])
def test_other_models(pos, frozen, bias):
    m = _plain_model(pos, bias, BF16, frozen)
    x = torch.randint(0, 512, (2, 128), generator=torch.Generator().manual_seed(3)).cuda()
    _steps_against_prefill(m, x, 110, 3e-2)


def test_trainable_patterns_decode():
    import supplement
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    supplement.enable(m)
    _steps_against_prefill(m, x, 120, 3e-2)


def test_split_route_model(monkeypatch):
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    monkeypatch.setattr(model_mod, "_FUSED", False)
    _steps_against_prefill(m, x, 120, 3e-2)


def test_generate():
    """Greedy tokens are the argmax of the whole-sequence forward over the same
    prefix (where its two best logits are further apart than both sides'
    rounding), and their log probabilities its log_softmax."""
    m = _plain_model(dtype=FP32, bias=False, frozen=(2,))
    x = torch.randint(0, 512, (3, 20), generator=torch.Generator().manual_seed(4)).cuda()
    counts = [20, 5, 13]
    tokens, logp = decode.generate(m, x, 12, counts)
    assert tokens.shape == logp.shape == (3, 12)
    for b, c in enumerate(counts):
        seq = torch.cat([x[b, :c], tokens[b]])[None]
        with torch.inference_mode():
            lg = m.forward_all_positions(seq)[0, c - 1:-1].double()
        lq = torch.log_softmax(lg, -1)
        best = lq.topk(2, -1)
        clear = best.values[:, 0] - best.values[:, 1] > 1e-4
        assert bool((best.indices[:, 0] == tokens[b])[clear].all()) and int(clear.sum()) >= 6
        got = lq.gather(1, tokens[b][:, None])[:, 0]
        assert bool(((got - logp[b].double()).abs() <= 1e-4).all())
    t0, l0 = decode.generate(m, x, 0)
    assert t0.shape == (3, 0) and l0.shape == (3, 0)


def test_inactive_sequences_and_reuse():
    m, _ = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    x = torch.randint(0, 50257, (2, 40), generator=torch.Generator().manual_seed(6)).cuda()
    cache = decode.PagedCache(m, 2, page_size=16, n_pages=6)
    a = decode.prefill(m, x, cache)
    cache.release(0)
    kept = [t.clone() for layer in cache.layers for t in layer if t is not None]
    tok = torch.tensor([3, 5]).cuda()
    lone = decode.decode_step(m, tok, cache)
    assert int(cache.lengths[0]) == 0 and int(cache.lengths[1]) == 41
    changed = sum(int((u != v).any()) for u, v in zip(kept, [t for layer in cache.layers for t in layer if t is not None]))
    assert changed > 0
    # sequence 1 goes on as it would in a batch of its own
    other = decode.PagedCache(m, 1, page_size=16)
    b = decode.prefill(m, x[1:], other)
    assert _rel(a[1], b[0]) <= 1e-2
    assert _rel(lone[1], decode.decode_step(m, tok[1:], other)[0]) <= 1e-2
    cache.release(1)
    assert len(cache._free) == 6
    c = decode.prefill(m, x, cache)
    assert _rel(c, a) <= 1e-2


def test_cache_refusals():
    m = _plain_model(frozen=(1,))
    x = torch.zeros(2, 20, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="block size"):
        decode.PagedCache(m, 2, max_length=129)
    cache = decode.PagedCache(m, 2, max_length=40, page_size=16, n_pages=4)
    with pytest.raises(ValueError, match="another batch size"):
        decode.prefill(m, x[:1], cache)
    with pytest.raises(ValueError, match="counts"):
        decode.prefill(m, x, cache, [20, 0])
    decode.prefill(m, x, cache, [20, 3])
    with pytest.raises(ValueError, match="empty sequences"):
        decode.prefill(m, x, cache)
    with pytest.raises(ValueError, match="exceed"):
        cache.reserve([21, 0])
    with pytest.raises(ValueError, match="used up"):
        cache.reserve([13, 30])
    assert cache._held == [20, 3]
    with pytest.raises(ValueError, match="one token per sequence"):
        decode.decode_step(m, x[0, :3], cache)
    m.transformer.h[0].attn.unfreeze_heads([1])
    with pytest.raises(RuntimeError, match="live heads changed"):
        decode.decode_step(m, x[0, :2], cache)


def test_graph_replays():
    """decode_tokens captured once and replayed with eager work between the
    replays: every replay's logits equal the eager step's."""
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    with torch.inference_mode():
        eager_cache, cache = decode.PagedCache(m, 1, page_size=16), decode.PagedCache(m, 1, page_size=16)
        decode.prefill(m, x[:, :60], eager_cache)
        decode.prefill(m, x[:, :60], cache)
        tok = x[0, 60:61].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        warm = decode.PagedCache(m, 1, page_size=16)
        decode.prefill(m, x[:, :60], warm)
        with torch.cuda.stream(side):
            warm.reserve(2)
            for _ in range(2):
                decode.decode_tokens(m, tok, warm)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = decode.decode_tokens(m, tok, cache)
        for i in range(8):                       # crosses a page boundary at 64
            tok.copy_(x[0, 60 + i:61 + i])
            want = decode.decode_step(m, x[0, 60 + i:61 + i], eager_cache)
            torch.cuda.synchronize()
            cache.reserve(1)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits, want), i
        assert int(cache.lengths[0]) == 68


def test_two_graphs_and_an_eager_call_share_nothing():
    """Split attention (workspace) in two captured graphs, replayed in turn
    with eager calls on another stream."""
    from decode_cases import paged_case, run_paged
    cs = [paged_case([4000 - 900 * i, 50], H=4, states=[0, 2, 0, 0], page=64, seed=20 + i) for i in range(2)]
    ms = [{n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()} for c in cs]
    for m in ms:
        m["_tables"] = (m["frozen"], m["hidx"], m["pidx"])

    def call(m):
        return kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], None, m["frozen"], m["hidx"],
                                       alpha=m["alpha"], rho=m["rho"], z=m["z"], validate=False)

    want = [call(m).clone() for m in ms]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in ms:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(m))
        graphs.append(g)
    side = torch.cuda.Stream()
    for rep in range(3):
        for i in (0, 1):
            graphs[i].replay()
            with torch.cuda.stream(side):
                eager = call(ms[1 - i])
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i]) and torch.equal(eager, want[1 - i])


def test_logprob_graph_forward_and_backward():
    """Few long rows (segments, workspace) with the backward, captured and
    replayed on new logits with eager work in between."""
    g = torch.Generator().manual_seed(9)
    xs = [(torch.randn(4, 140000, generator=g) * 2).to(BF16).cuda() for _ in range(3)]
    t = torch.randint(0, 140000, (4,), generator=g).cuda()
    x = xs[0].clone().requires_grad_()

    def loss_and_grad():
        r = kernel.token_logprobs(x, t, top=3, entropy=True)
        (gx,) = torch.autograd.grad(r.logp.sum() + 0.1 * r.entropy.sum(), x)
        return r.logp.detach(), r.top_index, gx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            loss_and_grad()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = loss_and_grad()
    for i in (0, 1, 2, 1):
        with torch.no_grad():
            x.copy_(xs[i])
        want = loss_and_grad()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


@pytest.mark.parametrize("view", [False, True])
def test_capture_is_refused_while_an_eager_graph_of_the_leaf_lives(view):
    """The refusal comes before anything is captured (the capture itself would
    end the process in torch's engine)."""
    x = torch.randn(2, 2, 1000, device="cuda") if view else torch.randn(4, 1000, device="cuda")
    x.requires_grad_()
    t = torch.zeros(x.shape[:-1], dtype=torch.long, device="cuda")
    alive = kernel.token_logprobs(x, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                # another stream, no capture: allowed
        kernel.token_logprobs(x, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            kernel.token_logprobs(x, t)
    torch.cuda.synchronize()
    assert torch.isfinite(alive.logp).all()
    del alive
    with torch.no_grad():                        # no gradient: nothing to refuse
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = kernel.token_logprobs(x, t)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(r.logp, kernel.token_logprobs(x.detach(), t).logp)


def test_training_loss_and_gradients():
    """-token_logprobs(...).logp.mean() against F.cross_entropy in float32
    (gradients of every parameter to fp32 rounding of a two-layer model)."""
    m = _plain_model(dtype=FP32, bias=False, frozen=(2,), T=64)
    m.train()
    g = torch.Generator().manual_seed(10)
    x, t = torch.randint(0, 512, (2, 64), generator=g).cuda(), torch.randint(0, 512, (2, 64), generator=g).cuda()
    t[0, :5] = -100
    ok = t != -100
    r = m.token_logprobs(x, t)
    (-r.logp.sum() / ok.sum()).backward()
    got = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    m.zero_grad()
    ref = torch.nn.functional.cross_entropy(m.forward_all_positions(x).flatten(0, 1), t.flatten())
    ref.backward()
    assert abs(float(-r.logp.detach().sum() / ok.sum()) - float(ref.detach())) <= 1e-5
    for n, p in m.named_parameters():
        if p.grad is not None:
            assert _rel(got[n], p.grad) <= 1e-4, n


def test_logits_of_a_step_feed_logprobs():
    """Decoded logits into alternatives: the top alternative is the argmax and
    its log probability the token's."""
    m, x = _small_model(T=128, layers=2, device="cuda", dtype=BF16)
    cache = decode.PagedCache(m, 1)
    logits = decode.prefill(m, x[:, :50], cache)
    best = logits.argmax(-1)
    r = kernel.token_logprobs(logits, best, top=5, entropy=True)
    assert float(r.logp[0]) == float(r.top_logp[0, 0])
    assert float(logits[0, r.top_index[0, 0]]) == float(logits[0, best[0]])
    assert float(r.entropy[0]) > 0
