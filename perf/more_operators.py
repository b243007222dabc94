"""The operators around the products and the attention of a training step, measured.

  embed      ``kernel.embed_tokens``: rows of an embedding by token, scaled, and
             the gradient of the whole embedding
  layernorm  ``kernel.add_layernorm``: a residual addition and its LayerNorm, and
             the gradients of the residual, the branch, the weight and the bias
  gelu8      ``kernel.gelu_packed``: the exact GELU that keeps its input for the
             backward pass in 8 bits, and the gradient that follows from them
  pack8      ``kernel.pack_activation`` / ``unpack_activation``: an activation
             into 8 bits with one power-of-two step per 32 channels, and back

``listed()`` holds the fixed cases, ``draw(rng)`` gives further ones of the same
ranges.  With ``own`` false ``run`` computes each operator in elementary torch
operations in float32; with ``own`` true it calls the framework.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32          # channels that share a step
IGNORE = -100       # tokens of padding


def _kernel():
    pkg = os.path.join(os.getcwd(), "selective-attention-freezing_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kernel
    return kernel


def listed():
    return [
        # the tokens of one decoding step of the 124M GPT: latency counts
        dict(name="embed_step", op="embed", dtype="bf16", wdtype="bf16", N=32, V=50304, C=768, scaled=False,
             train=False),
        # a training batch of the same model, float32 weights under bf16 activations
        dict(name="embed_train", op="embed", dtype="bf16", wdtype="fp32", N=16384, V=50304, C=768, scaled=False,
             train=True),
        # a long batch with the vocabulary and width of the Qwen-style model
        dict(name="embed_wide", op="embed", dtype="bf16", wdtype="bf16", N=32768, V=151936, C=896, scaled=True,
             train=True),
        # characters: every row of the embedding is used hundreds of times, odd sizes
        dict(name="embed_chars", op="embed", dtype="fp32", wdtype="fp32", N=16383, V=97, C=321, scaled=True, train=True),
        # one sub-layer's norm in a decoding step of the 124M GPT
        dict(name="layernorm_step", op="layernorm", dtype="bf16", res="bf16", wdtype="bf16", R=32, C=768, delta=True,
             bias=True, train=False),
        # a sub-layer of its training batch
        dict(name="layernorm_train", op="layernorm", dtype="bf16", res="bf16", wdtype="bf16", R=16384, C=768, delta=True,
             bias=True, train=True),
        # the 1B-class model, a float32 residual stream beside bf16 branches
        dict(name="layernorm_wide", op="layernorm", dtype="bf16", res="fp32", wdtype="fp32", R=8192, C=2048, delta=True,
             bias=False, train=True),
        # full precision, odd sizes, no addition
        dict(name="layernorm_odd", op="layernorm", dtype="fp32", res="fp32", wdtype="fp32", R=1023, C=1001, delta=False,
             bias=True, train=True),
        # the 1B-class model's MLP in a training batch: the most bytes
        dict(name="gelu8_train", op="gelu8", dtype="bf16", R=16384, C=8192),
        # a short sequence in full precision, the last block of each row is not full
        dict(name="gelu8_odd", op="gelu8", dtype="fp32", R=257, C=2001),
        # what the same model keeps of its hidden states
        dict(name="pack8_hidden", op="pack8", dtype="bf16", R=16384, C=2048),
        # a short sequence of odd width
        dict(name="pack8_odd", op="pack8", dtype="fp16", R=131, C=1999),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly widths that models have (multiples of 64), some odd ones."""
    c = _log_int(rng, lo, hi)
    return max(64, c // 64 * 64) if rng.random() < 0.6 else c


def draw(rng):
    """One more case: sizes spread over their logarithm, odd ones among them."""
    op = rng.choice(["embed", "embed", "layernorm", "layernorm", "gelu8", "pack8"])
    dt = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        C = _width(rng, 16, 4096)
        V = max(16, min(_log_int(rng, 50, 200000), 2 ** 27 // C))
        N = max(1, min(_log_int(rng, 1, 65536), 2 ** 25 // C))
        return dict(op=op, dtype=dt, wdtype=rng.choice([dt, "fp32"]), N=N, V=V, C=C, scaled=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    if op == "layernorm":
        C = _width(rng, 16, 8192)
        R = max(1, min(_log_int(rng, 1, 32768), 2 ** 24 // C))
        return dict(op=op, dtype=dt, res=rng.choice([dt, dt, "fp32"]), wdtype=rng.choice([dt, "fp32"]), R=R, C=C,
                    delta=rng.random() < 0.7, bias=rng.random() < 0.5, train=rng.random() < 0.7)
    C = _width(rng, 16, 16384)
    most = 2 ** 26 if dt == "fp32" else 2 ** 27
    if op == "pack8":
        most //= 4
    R = max(1, min(_log_int(rng, 1, 32768), most // C))
    return dict(op=op, dtype=dt, R=R, C=C)


# ---- inputs -------------------------------------------------------------------

def _odds(V):
    """Probabilities of the words of a vocabulary by rank: few are frequent."""
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    return p / p.sum()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, dtype=dt):
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=gen)

    op = case["op"]
    if op == "embed":
        N, V, C = case["N"], case["V"], case["C"]
        edge = _odds(V).cumsum(0).to(DEV)
        u = torch.empty(N, dtype=torch.float64, device=DEV).uniform_(0.0, 1.0, generator=gen)
        words = torch.randperm(V, generator=gen, device=DEV)
        tokens = words[torch.searchsorted(edge, u).clamp(max=V - 1)]
        tokens[torch.empty(N, device=DEV).uniform_(0.0, 1.0, generator=gen) < 0.02] = IGNORE
        weight = randn(V, C, std=0.02, dtype=DTYPES[case["wdtype"]])
        st = dict(case=case, tokens=tokens, weight=weight, scale=math.sqrt(C) if case["scaled"] else 1.0)
        if case["train"]:
            st["dy"] = randn(N, C, std=0.05)
            if own:
                weight.requires_grad_()
        return st
    R, C = case["R"], case["C"]
    if op == "layernorm":
        # a residual stream with some channels far from the others' size
        rt, wt = DTYPES[case["res"]], DTYPES[case["wdtype"]]
        size = torch.exp(torch.empty(C, device=DEV).normal_(0.0, 0.5, generator=gen))
        x = (randn(R, C, dtype=torch.float32) * size + 0.3).to(rt)
        st = dict(case=case, x=x, delta=randn(R, C, std=0.5) if case["delta"] else None,
                  weight=(1 + randn(C, std=0.2, dtype=torch.float32)).to(wt),
                  bias=randn(C, std=0.1, dtype=wt) if case["bias"] else None)
        if case["train"]:
            st["dy"] = randn(R, C, std=0.1)
            st["dr"] = randn(R, C, std=0.1, dtype=rt) if case["delta"] else None
            if own:
                for n in ("x", "delta", "weight", "bias"):
                    if st[n] is not None:
                        st[n].requires_grad_()
        return st
    # inputs of an activation: centred below zero, some rows larger than others
    rows = torch.exp(torch.empty(R, 1, device=DEV).normal_(0.0, 0.4, generator=gen))
    x = randn(R, C)
    x.mul_(rows.to(dt)).sub_(0.4)
    st = dict(case=case, x=x)
    if op == "gelu8":
        st["dy"] = randn(R, C, std=0.1)
        if own:
            x.requires_grad_()
    return st


# ---- the plain forms -------------------------------------------------------------

def _plain_embed(st):
    case, tok = st["case"], st["tokens"]
    skip = (tok < 0)[:, None]
    at = tok.clamp(min=0)
    y = (st["weight"][at].float() * st["scale"]).masked_fill(skip, 0.0).to(DTYPES[case["dtype"]])
    if not case["train"]:
        return y
    dy = st["dy"].float().masked_fill(skip, 0.0)
    dw = torch.zeros(case["V"], case["C"], device=DEV).index_add_(0, at, dy) * st["scale"]
    return y, dw.to(st["weight"].dtype)


def _plain_layernorm(st):
    case, w, b = st["case"], st["weight"].float(), st["bias"]
    r = st["x"] if st["delta"] is None else (st["x"].float() + st["delta"].float()).to(st["x"].dtype)
    x = r.float()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(d.square().mean(-1, keepdim=True) + 1e-5)
    xhat = d * rstd
    y = xhat * w
    if b is not None:
        y = y + b.float()
    out = [r, y.to(DTYPES[case["dtype"]])]
    if case["train"]:
        dy = st["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        if st["dr"] is not None:
            dx = dx + st["dr"].float()
        out.append(dx.to(r.dtype))
        if st["delta"] is not None:
            out.append(dx.to(st["delta"].dtype))
        out.append((dy * xhat).sum(0).to(st["weight"].dtype))
        if b is not None:
            out.append(dy.sum(0).to(b.dtype))
    return out


def _plain_packed(x):
    """float32 values that the 8 bits stand for: whole multiples, up to 127, of
    the step 2^(floor(log2 largest) - 6) of each block of channels."""
    R, C = x.shape
    pad = -C % BLOCK
    t = torch.nn.functional.pad(x.float(), (0, pad)).view(R, -1, BLOCK)
    e = ((t.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 6).clamp(min=0)
    step = torch.where(e > 0, e << 23, torch.full_like(e, 1 << 22)).view(torch.float32)
    return (torch.round(t / step).clamp(-127, 127) * step).view(R, -1)[:, :C]


def _plain_gelu8(st):
    x = st["x"].float()
    y = 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    u = _plain_packed(st["x"])
    slope = 0.5 * torch.erfc(u * -math.sqrt(0.5)) + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return y.to(st["x"].dtype), (st["dy"].float() * slope).to(st["x"].dtype)


# ---- the pass ----------------------------------------------------------------

def run(state):
    case = state["case"]
    op = case["op"]
    st = state
    if not own:
        if op == "pack8":
            return _plain_packed(st["x"]).to(st["x"].dtype)
        return {"embed": _plain_embed, "layernorm": _plain_layernorm, "gelu8": _plain_gelu8}[op](st)
    kernel = _kernel()
    if op == "embed":
        y = kernel.embed_tokens(st["tokens"], st["weight"], scale=st["scale"], ignore_index=IGNORE,
                                dtype=DTYPES[case["dtype"]])
        if not case["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, st["weight"], st["dy"])[0]
    if op == "layernorm":
        r, y = kernel.add_layernorm(st["x"], st["delta"], st["weight"], st["bias"], dtype=DTYPES[case["dtype"]])
        out = [r.detach(), y.detach()]
        if case["train"]:
            leaves = [st[n] for n in ("x", "delta", "weight", "bias") if st[n] is not None]
            heads, seeds = ((r, y), (st["dr"], st["dy"])) if st["dr"] is not None else ((y,), (st["dy"],))
            out += torch.autograd.grad(heads, leaves, seeds)
        return out
    if op == "gelu8":
        y = kernel.gelu_packed(st["x"])
        return y.detach(), torch.autograd.grad(y, st["x"], st["dy"])[0]
    return kernel.unpack_activation(kernel.pack_activation(st["x"]))


# ---- the definition in 64 bits ---------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "layernorm": _exact_layernorm, "gelu8": _exact_gelu8,
                "pack8": lambda c, s: _exact_packed(s["x"])}[case["op"]](case, st)


def _exact_embed(case, st):
    used = (st["tokens"] != IGNORE).nonzero()[:, 0]
    at = st["tokens"][used]
    y = torch.zeros(case["N"], case["C"], dtype=torch.float64, device=DEV)
    y[used] = st["weight"].index_select(0, at).double().mul_(st["scale"])
    if not case["train"]:
        return y
    # the rows of each word side by side, summed run by run
    order = torch.argsort(at, stable=True)
    words, count = torch.unique_consecutive(at[order], return_counts=True)
    g = st["dy"][used[order]].double() * st["scale"]
    dw = torch.zeros(case["V"], case["C"], dtype=torch.float64, device=DEV)
    dw[words] = torch.segment_reduce(g, "sum", lengths=count, axis=0) if len(words) else 0.0
    return y, dw


def _exact_layernorm(case, st):
    x = st["x"].detach().double()
    r = x if st["delta"] is None else x + st["delta"].detach().double()
    z = r.to(st["x"].dtype).double()               # the norm is that of the stored residual
    C = case["C"]
    m = z.sum(1) / C
    c = z - m[:, None]
    s = torch.sqrt(c.pow(2).sum(1) / C + 1e-5)
    n = c / s[:, None]
    w = st["weight"].detach().double()
    y = n * w
    if case["bias"]:
        y += st["bias"].detach().double()
    out = [r, y]
    if case["train"]:
        dy = st["dy"].double()
        h = dy * w
        dx = (h - (h.sum(1) / C)[:, None] - n * ((h * n).sum(1) / C)[:, None]) / s[:, None]
        if case["delta"]:
            dx += st["dr"].double()
        out.append(dx)
        if case["delta"]:
            out.append(dx)
        out.append((n * dy).sum(0))
        if case["bias"]:
            out.append(dy.sum(0))
    return out


def _exact_packed(x):
    x = x.detach().double()
    out = torch.empty_like(x)
    for c in range(0, x.size(1), BLOCK):
        b = x[:, c:c + BLOCK]
        top = b.abs().max(1).values
        step = torch.where(top > 0, torch.frexp(top).exponent - 1 - 6, -127).clamp(min=-127).long()
        step = ((step + 1023) << 52).view(torch.float64)[:, None]
        out[:, c:c + BLOCK] = torch.round(b / step).clamp(-127.0, 127.0) * step
    return out


def _exact_gelu8(case, st):
    def phi(t):
        return torch.special.erfc(t / -math.sqrt(2.0)) / 2

    x = st["x"].detach().double()
    y = x * phi(x)
    del x
    u = _exact_packed(st["x"])
    slope = phi(u) + u * torch.exp(u.square() / -2) / math.sqrt(2 * math.pi)
    return y, slope.mul_(st["dy"].double())


# ---- the least work ------------------------------------------------------------------

def work(case):
    es, C = SIZE[case["dtype"]], case["C"]
    if case["op"] == "embed":
        N, V, ws = case["N"], case["V"], SIZE[case["wdtype"]]
        rows = float((1 - (1 - _odds(V)).pow(0.98 * N)).sum())    # distinct words of a batch
        b, f = 8 * N + rows * C * ws + N * C * es, N * C
        if case["train"]:
            b += 0.98 * N * C * es + V * C * ws
            f += N * C
        return {"bytes": int(b), "flops": f}
    n = case["R"] * C
    if case["op"] == "layernorm":
        rs, ws = SIZE[case["res"]], SIZE[case["wdtype"]]
        vecs = C * ws * (2 if case["bias"] else 1)
        b, f = n * (rs + es) + vecs, 8 * n
        if case["delta"]:
            b += n * (es + rs)
        if case["train"]:
            # the residual again, dy (and dr), the gradients
            b += n * (2 * rs + es) + 2 * vecs
            f += 12 * n
            if case["delta"]:
                b += n * rs + (n * es if rs != es else 0)
        return {"bytes": b, "flops": f}
    held = n + case["R"] * ((C + BLOCK - 1) // BLOCK)
    if case["op"] == "pack8":
        return {"bytes": 2 * n * es + 2 * held, "flops": 4 * n}
    return {"bytes": 4 * n * es + 2 * held, "flops": 60 * n}
