"""Inputs and float64 references of the decoding operators' tests: paged
caches, single-token attention, appended tokens, token log probabilities.
Everything is made on the CPU; the references are plain loops over the
definitions."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def paged_case(lens, H=4, HKV=0, hd=64, page=16, dtype=torch.bfloat16, states=None, spare=2, seed=0, poison=True,
               patt_dtype=torch.float32, qscale=1.0, S=None):
    """A cache of ragged sequences: shuffled pages, NaN in every slot that
    holds no token, -1 in unused table entries; states per head 0 / 1 / 2."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    states = [0] * H if states is None else list(states)
    live = [h for h in range(H) if states[h] == 0]
    dense = [h for h in range(H) if states[h] == 1]
    n_tab = max(1, max((n + page - 1) // page for n in lens))
    pages = [(n + page - 1) // page for n in lens]
    P = sum(pages) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((B, n_tab), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n].int()
        at += n
    UK, HV = (HKV, HKV) if HKV else (len(live), H)

    def randn(*s):
        return torch.randn(*s, generator=g).to(dtype)

    kc, vc = randn(P, UK, page, hd), randn(P, HV, page, hd)
    if poison:
        held = torch.zeros(P, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for s in range(n):
                held[table[b, s // page], s % page] = True
        kc = kc.masked_fill(~held[:, None, :, None], float("nan"))
        vc = vc.masked_fill(~held[:, None, :, None], float("nan"))
    S = S or max(1, max(lens))
    alpha, rho = torch.randn(H, S, generator=g) * 0.5, torch.randn(H, S, generator=g) * 0.5
    z = torch.stack([torch.logsumexp(alpha[:, :n].double() + rho[:, :n].flip(1).double(), 1) for n in range(1, S + 1)],
                    1).float() if S <= 4096 else torch.zeros(H, S)
    if S > 4096:
        for n in lens:
            if n:
                z[:, n - 1] = torch.logsumexp(alpha[:, :n].double() + rho[:, :n].flip(1).double(), 1).float()
    hidx = torch.zeros(H, dtype=torch.int32)
    hidx[live] = torch.arange(len(live), dtype=torch.int32)
    pidx = torch.zeros(H, dtype=torch.int32)
    patt = None
    if dense:
        # rows in reverse order, so that pidx is no identity
        pidx[dense] = torch.arange(len(dense) - 1, -1, -1, dtype=torch.int32)
        p = torch.rand(len(dense), S, S, generator=g).tril()
        patt = (p / p.sum(-1, keepdim=True)).to(patt_dtype)
    return dict(q=randn(B, len(live), 1, hd) * qscale, kc=kc, vc=vc, table=table,
                lengths=torch.tensor(lens, dtype=torch.int32), frozen=torch.tensor(states, dtype=torch.int32), hidx=hidx,
                pidx=pidx, kvidx=(torch.arange(H, dtype=torch.int32) // (H // HKV)) if HKV else None, patt=patt,
                alpha=alpha, rho=rho, z=z, page=page, hd=hd)


def paged_reference(c, sm_scale=None):
    """(out, sum_j w_j |v_j|, lse) in float64, (B, H, hd), (B, H, hd), (B, H)."""
    H, hd, page = c["frozen"].numel(), c["hd"], c["page"]
    B = c["lengths"].numel()
    scale = hd ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(B, H, hd, dtype=torch.float64)
    mag = torch.zeros(B, H, hd, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    for b in range(B):
        n = int(c["lengths"][b])
        if n == 0:
            continue
        pos = torch.arange(n)
        pg, sl = c["table"][b].long()[pos // page], pos % page
        for h in range(H):
            kv = int(c["kvidx"][h]) if c["kvidx"] is not None else None
            v = c["vc"][pg, h if kv is None else kv, sl].double()
            st = int(c["frozen"][h])
            if st == 0:
                slot = int(c["hidx"][h])
                k = c["kc"][pg, slot if kv is None else kv, sl].double()
                s = (k @ c["q"][b, slot, 0].double()) * scale
                w = torch.softmax(s, 0)
                lse[b, h] = torch.logsumexp(s, 0) / math.log(2)
            elif st == 1:
                w = c["patt"][int(c["pidx"][h]), n - 1, :n].double()
            else:
                w = torch.exp(c["alpha"][h, :n].double() + c["rho"][h, :n].double().flip(0) - c["z"][h, n - 1].double())
            out[b, h] = w @ v
            mag[b, h] = w.abs() @ v.abs()
    return out, mag, lse


def paged_tolerance(c, ref, mag):
    """Elementwise bound of the operator's error.

    The output's own rounding is half a step of its type.  Before it, every
    weight is off by a relative d: the score's fp32 sum of hd products (relative
    (hd + 2) 2^-24 of sum |q k| scale, at most 2^-24 66 * 30 = 1.2e-4 of the
    weight at hd 64 and scores of size 30; the test scores stay below 10, head
    dims below 256), exp2 and the final division (a few 2^-23), and for 16-bit
    storage the two-term rounding of P (2^-16 bf16, 2^-22 fp16; fp16 weights
    below 2^-22 of the largest lose an absolute 2^-33).  2^-13 of sum w |v|
    covers these, in float32 2^-15 (the scores alone)."""
    dt = c["vc"].dtype
    d = 2.0 ** -15 if dt == torch.float32 else 2.0 ** -13
    floor = 0.0
    if dt == torch.float16:
        floor = float(c["lengths"].max()) * 2.0 ** -32 * float(torch.nan_to_num(c["vc"].float()).abs().max())
    return HALF_STEP[dt] * ref.abs() + d * mag + floor + 1e-30


def run_paged(kernel, c, dev="cuda", **kw):
    m = {n: (t.to(dev) if isinstance(t, torch.Tensor) else t) for n, t in c.items()}
    dec = bool((c["frozen"] == 2).any())
    return kernel.paged_mixed_attn(m["q"], m["kc"], m["vc"], m["table"], m["lengths"], m["patt"], m["frozen"], m["hidx"],
                                   m["pidx"], alpha=m["alpha"] if dec else None, rho=m["rho"] if dec else None,
                                   z=m["z"] if dec else None, kvidx=m["kvidx"], **kw)


def append_reference(x, weight, eps, cos, sin, pos):
    """norm and rotation in float64 of rows x (..., hd) at one position."""
    x = x.double()
    if weight is not None:
        x = weight.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if cos is not None:
        rd = cos.size(1)
        c, s = cos[pos].double(), sin[pos].double()
        y = x.clone()
        h = rd // 2
        y[..., :h] = x[..., :h] * c[:h] - x[..., h:rd] * s[:h]
        y[..., h:rd] = x[..., h:rd] * c[h:] + x[..., :h] * s[h:]
        x = y
    return x


def logprob_reference(logits, tokens, top, scale, ignore=-100):
    """(logp, entropy, top indices, top logp, log softmax) in float64 on the CPU."""
    x = logits.double() * scale
    lq = x - torch.logsumexp(x, -1, keepdim=True)
    p = lq.exp()
    ent = -(p * lq.clamp(min=-1e30)).nan_to_num(nan=float("nan")).sum(-1)
    R, V = x.shape
    logp = torch.zeros(R, dtype=torch.float64)
    for r in range(R):
        t = int(tokens[r])
        if t != ignore:
            logp[r] = lq[r, t] if 0 <= t < V else float("nan")
    idx = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    return logp, ent, idx, lq.gather(1, idx), lq
