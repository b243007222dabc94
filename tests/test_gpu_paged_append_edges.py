"""Arguments of paged_append_ at the edge of what it documents."""
import pytest
import torch

import kernel
from test_gpu_paged_append import _case, _run

pytestmark = pytest.mark.gpu


def _dev(c):
    return {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in c.items()}


def test_leading_dims_of_the_rotary_caches():
    """Singleton ones are dropped, of each cache on its own; a cache per
    sequence is refused, not read as one long cache."""
    c = _case(T=3, starts=(0, 5), seed=1)
    want = _run(c)

    def call(cos, sin):
        d = _dev(c)
        q = kernel.paged_append_(d["k"], d["v"], d["kc"], d["vc"], d["table"], d["positions"], q=d["q"], cos=cos, sin=sin,
                                 q_weight=d["qw"], k_weight=d["kw"], eps=1e-5)
        return q, d["kc"], d["vc"]

    cos, sin = c["cos"].cuda(), c["sin"].cuda()
    for a, b in ((cos[None, None], sin[None, None]), (cos, sin[None]), (cos[None], sin)):
        assert all(torch.equal(x, y) for x, y in zip(call(a, b), want))
    for a, b in ((cos.expand(2, -1, -1), sin.expand(2, -1, -1)), (cos, sin.expand(2, 1, -1, -1)), (cos.expand(2, -1, -1), sin)):
        with pytest.raises(ValueError, match="leading singleton"):
            call(a, b)
    with pytest.raises(ValueError):
        call(cos[0], sin[0])


def test_values_without_heads():
    """Refused: q rows would come back unwritten."""
    d = _dev(_case(T=3, seed=2))
    with pytest.raises(ValueError, match="v and v_cache are required"):
        kernel.paged_append_(None, d["v"][:, :0], None, d["vc"][:, :0], d["table"], d["positions"], q=d["q"])
    for shape in ((0, 2, 3, 64), (2, 2, 0, 64)):
        v = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        q = kernel.paged_append_(v, v, d["kc"], d["vc"], d["table"][:shape[0]], d["positions"][:shape[0]], q=v)
        assert q.shape == shape
