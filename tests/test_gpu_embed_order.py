"""The order in which an embedding's gradient adds up, as its documentation states it,
bit by bit: the same additions in float32 on the CPU."""
import numpy as np
import pytest
import torch

import kernel
from train_cases import DEV, rnd

pytestmark = pytest.mark.gpu


def _chunk(N, C):
    waves = -(-N // 64) * -(-C // 256)
    return 64 if waves >= 1024 else 32 if waves >= 512 else 16


def _in_order(rows):
    acc = np.zeros_like(rows[0])
    for r in rows:
        acc = acc + r
    return acc


def _reference(tokens, dy, V, scale):
    """Positions sorted by word and cut into chunks: each chunk's part of a word in the
    order of its positions; a word of several chunks has its first part and every
    sixteenth of the others in the first of 16 runs, and the runs are added in order."""
    N, C = dy.shape
    order = np.argsort(tokens, kind="stable")
    size = _chunk(N, C) if N > 64 else N
    dw = np.zeros((V, C), np.float32)
    for v in range(V):
        at = np.flatnonzero(tokens[order] == v)
        if not len(at):
            continue
        parts = [_in_order(dy[order[at[at // size == k]]]) for k in range(at[0] // size, at[-1] // size + 1)]
        first, rest = parts[0], parts[1:]
        runs = [_in_order(([first] if l == 0 else []) + rest[l::16] or [np.zeros(C, np.float32)]) for l in range(16)]
        dw[v] = _in_order(runs) * np.float32(scale)
    return dw


@pytest.mark.parametrize("N,V,C", [(64, 3, 9), (65, 3, 9), (700, 2, 5), (5000, 7, 5), (9001, 40, 33), (20000, 5, 4), (40000, 3, 5),
                                   (34000, 9, 260)])
def test_order(N, V, C):
    """One chunk, few and many, of 16, 32 and 64 positions, every way of sorting."""
    g = torch.Generator(device=DEV).manual_seed(N)
    tokens = (torch.rand(N, device=DEV, generator=g) ** 2 * V).long().clamp(max=V - 1)
    w, dy = torch.zeros(V, C, device=DEV, requires_grad=True), rnd(N, C, seed=N + 1)
    (dw,) = torch.autograd.grad(kernel.embed_tokens(tokens, w, scale=1.7), w, dy)
    want = _reference(tokens.cpu().numpy(), dy.cpu().numpy(), V, 1.7)
    assert np.array_equal(dw.cpu().numpy(), want)
