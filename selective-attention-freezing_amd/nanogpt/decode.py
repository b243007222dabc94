"""Decoding with the GPT of ``nanogpt.model``: a paged cache, the step of one
token per sequence, and greedy generation.

    cache = PagedCache(model, batch=4)
    logits = prefill(model, prompts, cache, counts)      # (4, vocab), ragged prompts right-padded
    logits = decode_step(model, tokens, cache)           # (4, vocab)
    tokens, logp = generate(model, prompts, 64, counts)

Each layer keeps the keys of its live heads only (frozen heads have none) and
every head's values, in pages that all layers address through one page table
(``kernel.paged_append_``, ``kernel.paged_mixed_attn``).  Which heads are live is
part of the cache's layout: freezing or unfreezing heads afterwards makes the
cache unusable (checked at each call).  Inference only.

``decode_tokens`` is the device half of ``decode_step``: it reads no host state,
so it can be captured into a HIP graph; ``cache.reserve(1)`` before each replay
provides the pages, and after a change of weights or trainable patterns
``cache.check(model)`` what the step derives from them.  A step captured before
other heads were frozen has to be captured again.
"""
import torch

import kernel as _kernel_mod


class PagedCache:
    """Pages for `batch` sequences of up to max_length tokens (default: the
    model's block size).  n_pages bounds the pool (default: enough for every
    sequence at max_length); page_size is a power of two, at least 16."""

    def __init__(self, model, batch, max_length=None, page_size=64, n_pages=None):
        cfg = model.config
        max_length = cfg.block_size if max_length is None else int(max_length)
        if not 0 < max_length <= cfg.block_size:
            raise ValueError(f"max_length must be between 1 and the model's block size {cfg.block_size}")
        per_seq = -(-max_length // page_size)
        n_pages = batch * per_seq if n_pages is None else int(n_pages)
        p = model.lm_head.weight
        dev, dt, hd = p.device, p.dtype, cfg.n_embd // cfg.n_head
        self.max_length, self.page_size = max_length, page_size
        self.layers, self._live, self._seen = [], [], []
        for attn in model.attn_modules():
            live = self._live_heads(attn)
            kc = torch.empty(n_pages, len(live), page_size, hd, device=dev, dtype=dt) if live else None
            self.layers.append((kc, torch.empty(n_pages, cfg.n_head, page_size, hd, device=dev, dtype=dt)))
            self._live.append(live)
            self._seen.append(attn._uf_idx)
        self.page_table = torch.full((batch, per_seq), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.active = torch.ones(batch, dtype=torch.int32, device=dev)
        # (positions, hd) rows, as paged_append_ takes them
        self.rope = tuple(t[0, 0] for t in model.rotary(cfg.block_size, dt)) if model.rotary is not None else None
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch)]
        self._held = [0] * batch    # tokens that pages are reserved for
        self._on = [True] * batch

    @staticmethod
    def _live_heads(attn):
        if attn._fz_dirty:
            attn._refresh_freeze_cache()
        return attn._uf_idx.tolist()

    def check_heads(self, model):
        """Raise if the model's live heads are not the cache's."""
        # a refresh of a layer's freeze tables, here or in another forward, makes
        # a new _uf_idx: only then are its heads read back
        for i, attn in enumerate(model.attn_modules()):
            if attn._fz_dirty or attn._uf_idx is not self._seen[i]:
                if self.lengths.is_cuda and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("heads were frozen or unfrozen: call PagedCache.check(model) before the capture")
                if self._live_heads(attn) != self._live[i]:
                    raise RuntimeError("the model's live heads changed since the cache was made")
                self._seen[i] = attn._uf_idx

    def check(self, model):
        """check_heads(), and what a step keeps of the model's weights, freeze
        states and trainable patterns brought up to date."""
        self.check_heads(model)
        for attn in model.attn_modules():
            attn.prepare_step()

    def reserve(self, new):
        """Pages for `new` more tokens of every active sequence (a number, or
        one per sequence); the page table is written only when pages are
        added.  Raises, changing nothing, if a sequence or the pool is full."""
        batch = len(self._held)
        new = [int(new)] * batch if not hasattr(new, "__len__") else [int(n) for n in new]
        if len(new) != batch or min(new) < 0:
            raise ValueError("one non-negative token count per sequence is required")
        want = [h + (n if on else 0) for h, n, on in zip(self._held, new, self._on)]
        if max(want) > self.max_length:
            raise ValueError(f"a sequence would exceed the cache's {self.max_length} tokens")
        add = [-(-w // self.page_size) - len(p) for w, p in zip(want, self._pages)]
        if sum(add) > len(self._free):
            raise ValueError(f"the cache's pages are used up ({sum(add)} needed, {len(self._free)} free)")
        rows = []
        for b, n in enumerate(add):
            for _ in range(n):
                self._pages[b].append(self._free.pop())
            if n:
                rows.append(b)
        self._held = want
        for b in rows:
            ids = torch.tensor(self._pages[b], dtype=torch.int32)
            self.page_table[b, :len(ids)].copy_(ids)

    def _back_to(self, held, on):
        """Undo reservations: the sequences hold `held` tokens again."""
        self._held, self._on = held, on
        for b, pages in enumerate(self._pages):
            keep = -(-held[b] // self.page_size)
            if len(pages) > keep:
                self._free += reversed(pages[keep:])
                del pages[keep:]
                self.page_table[b, keep:].fill_(-1)

    def release(self, b):
        """Give back sequence b's pages; it becomes empty and inactive."""
        self._free += self._pages[b]
        self._pages[b] = []
        self._held[b] = 0
        self._on[b] = False
        self.page_table[b].fill_(-1)
        self.lengths[b] = 0
        self.active[b] = 0


@torch.no_grad()
def prefill(model, idx, cache, counts=None):
    """Run prompts idx (B, T), right-padded (with any numbers) where counts
    (B,) are smaller than T, from empty sequences; returns each prompt's
    next-token logits (B, vocab).  A call that raises leaves them empty."""
    B, T = idx.shape
    cache.check(model)
    counts = [T] * B if counts is None else [int(c) for c in counts]
    if len(counts) != len(cache._held) or len(counts) != B:
        raise ValueError("the cache was made for another batch size")
    if any(cache._held):
        raise ValueError("prefill starts from empty sequences (PagedCache.release)")
    if not 1 <= min(counts) or max(counts) > T:
        raise ValueError("counts must lie between 1 and the prompts' width")
    if T > model.config.block_size:
        raise ValueError(f"prompts of {T} tokens exceed the model's block size {model.config.block_size}")
    on = cache._on
    try:
        cache._on = [True] * B
        cache.reserve(counts)
        n = torch.tensor(counts, dtype=torch.int32, device=idx.device)
        start = torch.zeros_like(n)

        def sink(layer):
            kc, vc = layer
            return lambda k, v: _kernel_mod.paged_append_(k, v, kc if k is not None else None, vc, cache.page_table, start,
                                                          n)

        if min(counts) < T:   # token 0 stands for the padding, which need not be one
            idx = torch.where(torch.arange(T, device=idx.device) < n[:, None], idx, 0)
        h = model.forward_hidden(idx, [sink(layer) for layer in cache.layers])
        logits = model.lm_head(h[torch.arange(B, device=idx.device), (n - 1).long()])
    except BaseException:
        cache._back_to([0] * B, on)
        raise
    cache.lengths.copy_(n)
    cache.active.fill_(1)
    return logits


@torch.no_grad()
def decode_tokens(model, tokens, cache):
    """The device half of decode_step (pages are reserved by the caller)."""
    cache.check_heads(model)
    if tokens.numel() != len(cache._held):
        raise ValueError("one token per sequence of the cache is required")
    tr = model.transformer
    pos = cache.lengths
    lengths = pos + cache.active
    # an inactive sequence's token may be anything: token 0 stands for it
    x = tr.wte(torch.where(cache.active > 0, tokens.reshape(-1), 0)[:, None])
    if model.rotary is None:
        x = x + tr.wpe(pos.long().clamp(max=model.config.block_size - 1))[:, None]
    fused = x.dtype in (torch.bfloat16, torch.float16) and x.size(-1) <= 2048
    x = x.contiguous()

    def norm(delta, ln):
        # x += delta, then its LayerNorm
        if fused:
            return _kernel_mod.add_layernorm_(x, delta, ln.weight, ln.bias)
        if delta is not None:
            x.add_(delta)
        return ln(x)

    h = norm(None, tr.h[0].ln_1)
    for i, block in enumerate(tr.h):
        attn, mlp = block.attn, block.mlp
        y = attn.attend_cached(h, (*cache.layers[i], cache.page_table), pos, lengths, cache.active, cache.rope)
        h = norm(attn.c_proj(y), block.ln_2)
        h = norm(mlp(h), tr.h[i + 1].ln_1 if i + 1 < len(tr.h) else tr.ln_f)
    logits = model.lm_head(h[:, 0])
    cache.lengths.copy_(lengths)
    return logits


def decode_step(model, tokens, cache):
    """Append tokens (B,) to the sequences (inactive ones ignore theirs) and
    return the next tokens' logits (B, vocab).  A call that raises leaves the
    sequences as they were."""
    held = cache._held
    try:
        cache.reserve(1)
        return decode_tokens(model, tokens, cache)
    except BaseException:
        cache._back_to(held, cache._on)
        raise


@torch.no_grad()
def generate(model, idx, max_new_tokens, counts=None, cache=None):
    """Greedy continuation of prompts idx (B, T), right-padded where counts
    (B,) are smaller than T: (tokens (B, n) int64, their log probabilities
    (B, n) fp32)."""
    B = idx.size(0)
    if cache is None:
        most = idx.size(1) if counts is None else max(int(c) for c in counts)
        cache = PagedCache(model, B, max_length=min(model.config.block_size, most + max_new_tokens))
    logits = prefill(model, idx, cache, counts)
    tokens, logps = [], []
    ignored = torch.full((B,), -100, dtype=torch.int64, device=idx.device)
    for i in range(max_new_tokens):
        r = _kernel_mod.token_logprobs(logits, ignored, top=1)
        tokens.append(r.top_index[:, 0])
        logps.append(r.top_logp[:, 0])
        if i + 1 < max_new_tokens:
            logits = decode_step(model, tokens[-1], cache)
    if not tokens:
        return idx.new_zeros(B, 0), torch.zeros(B, 0, device=idx.device)
    return torch.stack(tokens, 1), torch.stack(logps, 1)
