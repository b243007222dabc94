"""The training operators in captured graphs, on other streams and in several
threads: the eager results, bit by bit, replay after replay."""
import threading

import pytest
import torch

import kernel
from train_cases import BF16, DEV, F32, rnd

pytestmark = pytest.mark.gpu


def _embed(seed, N=9000, V=700, C=96):
    t = torch.randint(0, V, (N,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))
    return [rnd(V, C, seed=seed, dtype=BF16)], lambda w: [kernel.embed_tokens(t, w, scale=2.0)], [rnd(N, C, seed=seed + 1, dtype=BF16)]


def _norm(seed, R=5000, C=200):
    leaves = [rnd(R, C, seed=seed), rnd(R, C, seed=seed + 1, dtype=BF16), rnd(C, seed=seed + 2), rnd(C, seed=seed + 3)]
    return leaves, lambda *a: list(kernel.add_layernorm(*a)), [rnd(R, C, seed=seed + 4), rnd(R, C, seed=seed + 5, dtype=BF16)]


def _gelu(seed, R=300, C=1000):
    return [rnd(R, C, seed=seed, dtype=BF16)], lambda x: [kernel.gelu_packed(x)], [rnd(R, C, seed=seed + 1, dtype=BF16)]


def _mlp(seed, R=4000, C=64, bias=True):
    x, w1, w2 = rnd(R, C, seed=seed, dtype=BF16), rnd(256, C, seed=seed + 1, dtype=BF16), rnd(C, 256, seed=seed + 2, dtype=BF16)
    b = [rnd(256, seed=seed + 3, dtype=BF16), rnd(C, seed=seed + 4, dtype=BF16)] if bias else []
    return [x, w1, w2, *b], lambda *a: [kernel.mlp_packed(*a)], [rnd(R, C, seed=seed + 5, dtype=BF16)]


def _together(seed, B=3, T=500, V=333, C=64):
    """Embedding, norms, MLP and loss in one run, as a training pass has them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, nxt = (torch.randint(0, V, (B, T), device=DEV, generator=g) for _ in range(2))
    leaves = [rnd(V, C, seed=seed, dtype=BF16, std=0.5), rnd(4 * C, C, seed=seed + 1, dtype=BF16, std=0.1),
              rnd(C, 4 * C, seed=seed + 2, dtype=BF16, std=0.1), rnd(C, seed=seed + 3), rnd(C, seed=seed + 4)]

    def run(wte, fc, proj, w, b):
        x = kernel.embed_tokens(t, wte)
        _, h = kernel.add_layernorm(x, None, w, b)
        x, h = kernel.add_layernorm(x, kernel.mlp_packed(h, fc, proj), w, b)
        _, h = kernel.add_layernorm(x, kernel.gelu_packed(h), w, b)
        return [kernel.token_logprobs(torch.nn.functional.linear(h, wte), nxt).logp]

    return leaves, run, [torch.full((B, T), -1.0 / (B * T), device=DEV)]


CASES = dict(embed=_embed, embed_counted=lambda seed: _embed(seed, N=20000, C=40), norm=_norm, gelu=_gelu, mlp=_mlp, together=_together)


def _eager(leaves, run, seeds):
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    out = run(*leaves)
    return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, seeds))


def _junk():
    """Whatever the allocator has free, in use with other values."""
    return [torch.full((n,), 9e3, device=DEV) for n in (1 << 9, 1 << 14, 1 << 17, 1 << 20) for _ in range(3)]


@pytest.mark.parametrize("name", sorted(CASES))
def test_captured(name):
    """Two graphs of one operator, replayed in turn with eager work between, on
    changing inputs."""
    first = CASES[name](1)
    graphs = []
    for _ in range(2):
        leaves = [t.detach().clone().requires_grad_() for t in first[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                out = first[1](*leaves)
                torch.autograd.grad(out, leaves, first[2])
                del out
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = first[1](*leaves)
            got = [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, first[2]))
        del out
        graphs.append((graph, leaves, got))
    base = [t.detach().clone() for t in first[0]]
    for i in range(4):
        for graph, leaves, got in graphs:
            with torch.no_grad():
                for t, b in zip(leaves, base):
                    t.copy_(b * (1 + 0.25 * (i % 2)))
            held = _junk()
            expect = _eager([t.detach() for t in leaves], first[1], first[2])
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, expect):
                assert torch.equal(a, b), (name, i)
            assert held


@pytest.mark.parametrize("name", sorted(CASES))
def test_capture_is_refused_while_an_eager_graph_lives(name):
    leaves, run, seeds = CASES[name](2)
    leaves = [t.requires_grad_() for t in leaves]
    alive = run(*leaves)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run(*leaves)
    torch.cuda.synchronize()
    assert all(torch.isfinite(t).all() for t in alive)
    # without a gradient there is nothing to refuse
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        got = run(*leaves)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, alive):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", sorted(CASES))
def test_other_streams(name):
    """Two calls at once on streams of their own, behind long work of their
    inputs' stream, with the backward passes beside each other."""
    make = CASES[name]
    cases = [make(5), make(6)]
    want = [_eager(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        busy = rnd(2048, 2048, seed=1)
        for _ in range(10):
            busy = busy @ busy * 1e-3
        slow = [[t.detach() + 0 for t in c[0]] for c in cases]
        got = []
        for c, ts, s in zip(cases, slow, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_eager(ts, c[1], c[2]))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)


def test_threads():
    cases = [make(7 + i) for i, make in enumerate((_embed, _norm, _gelu, _embed))]
    want = [_eager(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(c, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = _eager(*c)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, w))
        except BaseException as e:   # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_together_in_float32():
    """Finite and the same bits again; test_gpu_train_model compares such a run."""
    leaves, run, seeds = _together(9)
    leaves = [t.to(F32) for t in leaves]
    got = _eager(leaves, run, seeds)
    assert all(torch.isfinite(t).all() for t in got)
    again = _eager(leaves, run, seeds)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
