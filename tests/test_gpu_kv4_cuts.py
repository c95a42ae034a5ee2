"""GPU tests of how the pages of a 4-bit cache are cut among workgroups: tile groups in
parts of their own, even cuts through many groups, long rows in many parts, more groups
than workgroups.  Oracle and bounds are those of test_gpu_kv4."""

import numpy as np
import pytest
import torch

from oracle import kv4 as O
from test_gpu_kv4 import attention_inputs, check_attention, contents, ints, say

pytestmark = pytest.mark.gpu

CUTS = [
    # B, T, HQ, H, D, pages, block, lengths
    (70, 2, 4, 4, 64, 5, "causal", [(37 * b) % 300 for b in range(70)]),      # more sequences than a wave has lanes
    (66, 1, 2, 1, 128, 40, "causal", [2500 if b == 65 else b for b in range(66)]),   # one long among short ones
    (130, 1, 8, 8, 64, 2, "causal", [(5 * b) % 127 for b in range(130)]),     # over a thousand groups of a page or two
    (1, 1, 1, 1, 64, 600, "causal", [38390]),                                # one row in as many parts as there may be
    (2, 3, 2, 2, 128, 130, "causal", [8300, 3]),                              # parts of one group beside a group of one page
    (3, 169, 64, 8, 128, 3, "none", [2, 0, 1]),                               # more tile groups than workgroups, one page each
    (10, 128, 16, 4, 64, 10, "causal", [0, 500, 3, 64, 511, 200, 1, 128, 300, 77]),  # row tiles over unequal lengths
    (1, 17, 4, 4, 64, 17, "causal", [1070]),                                  # a page more than a part begins with
]


@pytest.mark.parametrize("B,T,HQ,H,D,pages,block,lengths", CUTS)
def test_attention_of_any_cut(pkg, dev, B, T, HQ, H, D, pages, block, lengths):
    say("attention cut", B, T, HQ, H, D, pages)
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, "bf16", block, lengths, None, seed=B + T)
    n = ints(lengths, dev)
    out, lse = pkg.kv4_attention(q.to(dev), cache, n, block=block)
    again, _ = pkg.kv4_attention(q.to(dev), cache, n, block=block)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    check_attention(cache, q, "bf16", block, lengths, None, None, D ** -0.5, out, lse)


@pytest.mark.parametrize("B,T,HQ,H,D,pages,block,lengths", CUTS)
def test_weights_of_any_cut(pkg, dev, B, T, HQ, H, D, pages, block, lengths):
    say("weights cut", B, T, HQ, H, D, pages)
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, "bf16", block, lengths, None, seed=B + T)
    n = ints(lengths, dev)
    _, lse = pkg.kv4_attention(q.to(dev), cache, n, block=block)
    w = torch.rand(B, H, cache.slots, generator=torch.Generator().manual_seed(8)) * 3
    got = pkg.kv4_weights(q.to(dev), cache, n, lse, w.to(dev), block=block)
    torch.cuda.synchronize()
    K, _ = contents(cache)
    ref, added, mass = O.weights(q.double().numpy(), K, lengths, [T] * B, [T] * B, block, D ** -0.5,
                                 lse.double().cpu().numpy(), w.double().numpy(), None)
    tol = added * (mass[..., None] * 2.0 ** -16 + 2.0 ** -18) + ref * 2.0 ** -20
    assert np.all(np.abs(got.double().cpu().numpy() - ref) <= tol)


@pytest.mark.parametrize("n,keep", [(700, 301), (17000, 4099)])
def test_evict_takes_weights_at_any_float(pkg, dev, n, keep):
    """Weights that begin at no whole 16 bytes, rows of an odd budget: as from an aligned copy."""
    say("evict alignment", n, keep)
    H, D, pages = 3, 64, (n + 63) // 64
    made = []
    g = torch.Generator().manual_seed(n)
    w = torch.rand(H * pages * 64, generator=g)
    data = torch.randint(0, 256, (pages, H, O.page_bytes(D)), generator=g, dtype=torch.uint8)
    table = torch.randperm(pages, generator=g).view(1, pages).int()
    for off in (0, 1, 3):
        cache = pkg.KV4Cache(data.to(dev), table.to(dev), D)
        wd = torch.zeros(w.numel() + 8, device=dev)[off:off + w.numel()].copy_(w.to(dev)).view(1, H, pages * 64)
        made.append((*pkg.kv4_evict(cache, ints([n], dev), wd, keep, 5), cache.data))
    torch.cuda.synchronize()
    for other in made[1:]:
        for x, y in zip(other, made[0]):
            assert torch.equal(x, y)
    for h in range(H):
        ref = O.evict(w.view(H, -1)[h, :n].double().numpy(), n, keep, 5)
        assert np.array_equal(made[0][2][0, h].cpu().numpy(), ref)
