"""Offsets past 32 bits: pages at the end of caches of more than 2^32 elements,
and rows at the end of logits of more than 2^32 bytes."""
import pytest
import torch

import kernel
from decode_cases import logprob_reference, paged_case, paged_reference, paged_tolerance, run_paged

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _spread(c, P):
    """The case's pages at the start, in the middle and at the end of pools of
    P pages (whose other pages hold whatever is there)."""
    n = c["kc"].size(0)
    where = torch.linspace(0, P - 1, n).long()
    pools = []
    for t in (c["kc"], c["vc"]):
        pool = torch.empty((P, *t.shape[1:]), dtype=t.dtype, device="cuda")
        pool[where.cuda()] = t.cuda()
        pools.append(pool)
    table = torch.where(c["table"] >= 0, where[c["table"].clamp(min=0).long()].int(), -1)
    return pools[0], pools[1], table.cuda()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("lens", [[70, 200, 33], [3000, 40, 900]])
def test_caches(lens, dtype):
    """Attention and append, whole sequences and key ranges."""
    c = paged_case(lens, H=16, HKV=8, hd=128, dtype=dtype, page=64, states=[0, 2] * 8, seed=lens[0])
    kc, vc, table = _spread(c, (1 << 32) // (8 * 64 * 128) + 300)
    assert vc.numel() > 1 << 32
    m = {n: (t.cuda() if isinstance(t, torch.Tensor) and n not in ("kc", "vc", "table") else t) for n, t in c.items()}
    out = kernel.paged_mixed_attn(m["q"], kc, vc, table, m["lengths"], None, m["frozen"], m["hidx"], alpha=m["alpha"],
                                  rho=m["rho"], z=m["z"], kvidx=m["kvidx"])
    ref, mag, _ = paged_reference(c)
    assert bool(((out.double().cpu()[:, :, 0] - ref).abs() <= paged_tolerance(c, ref, mag)).all())
    # each sequence's last token written again, with other values
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(3, 8, 1, 128, generator=g).to(dtype) for _ in range(2))
    kernel.paged_append_(k.cuda(), v.cuda(), kc, vc, table, m["lengths"] - 1)
    for b, n in enumerate(lens):
        pg, sl = int(c["table"][b, (n - 1) // 64]), (n - 1) % 64
        c["kc"][pg, :, sl], c["vc"][pg, :, sl] = k[b, :, 0], v[b, :, 0]
    out = kernel.paged_mixed_attn(m["q"], kc, vc, table, m["lengths"], None, m["frozen"], m["hidx"], alpha=m["alpha"],
                                  rho=m["rho"], z=m["z"], kvidx=m["kvidx"])
    ref, mag, _ = paged_reference(c)
    assert bool(((out.double().cpu()[:, :, 0] - ref).abs() <= paged_tolerance(c, ref, mag)).all())


@pytest.mark.parametrize("V,dtype", [(200003, FP16), (1000, BF16)])
def test_logits(V, dtype):
    """Rows at the end, with their gradient (2^-17 of log V and half a step, as
    test_gpu_token_logprobs.py derives them)."""
    R = (1 << 32) // V + 5
    x = torch.empty(R, V, dtype=dtype, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    t = torch.zeros(R, dtype=torch.long, device="cuda")
    t[-3:] = torch.tensor([5, V - 1, 77], device="cuda")
    x.requires_grad_()
    r = kernel.token_logprobs(x, t, top=3, entropy=True)
    g = torch.zeros(R, device="cuda")
    g[-3:] = torch.tensor([1.0, -0.5, 2.0], device="cuda")
    (dx,) = torch.autograd.grad(r.logp, x, g)
    tail, tt = x.detach()[-3:].cpu(), t[-3:].cpu()
    logp, ent, idx, tlp, lq = logprob_reference(tail, tt, 3, 1.0)
    for got, want in ((r.logp, logp), (r.entropy, ent), (r.top_logp, tlp)):
        assert bool(((got[-3:].detach().double().cpu() - want).abs() <= 2.0 ** -17 * 13).all())
    assert torch.equal(r.top_index[-3:].cpu(), idx)
    want = -g[-3:].cpu().double()[:, None] * lq.exp()
    want[torch.arange(3), tt] += g[-3:].cpu().double()
    step = 2.0 ** -8 if dtype == BF16 else 2.0 ** -11
    assert bool(((dx[-3:].double().cpu() - want).abs() <= (step + 2.0 ** -15) * want.abs() + 2.0 ** -25 + 1e-30).all())
    assert bool((dx[:-3][::997] == 0).all())
