"""GPU tests of the 8-bit cache's attention at the bound that weights in two parts allow (2^-17 of each).

The bound is oracle.kv8.output_range with `parts` of 2; test_oracle_kv8_weights shows on the CPU that one f16
part lies outside of it.
"""

import numpy as np
import pytest
import torch

from oracle import kv8 as O
from test_gpu_kv8 import ATTENTION, attention_64, attention_inputs, contents, ints, same, say
from test_gpu_kv8_tiles import check

pytestmark = pytest.mark.gpu


def outside(cache, q, lengths, counts, block, masks, window, sinks, out, lse, dtype, parts):
    """How many outputs lie outside of the bound; the logarithms of the sums have to be within theirs."""
    B, T, HQ, D = q.shape
    c = [T] * B if counts is None else counts
    bad = 0
    for b, (ro, rl, weight, mass) in enumerate(attention_64(cache, q, lengths, c, block, masks, window, sinks)):
        err = mass * 2.0 ** -16
        got, f = lse[b].double().view(rl.shape), rl > -float("inf")
        assert torch.equal(f, got > -float("inf"))
        assert torch.all((got - rl)[f].abs() <= (err + 2.0 ** -20 * (1 + rl.abs()))[f]), b
        # two bf16 parts have a weight's whole range, whatever the row's largest one is
        lo, hi = O.output_range(ro.cpu().numpy(), weight.cpu().numpy(), err.cpu().numpy(), dtype, 0.0, parts)
        o = out[b].double().view(ro.shape).cpu().numpy()
        bad += int(((o < lo) | (o > hi)).sum())
    return bad


@pytest.mark.parametrize("sharp,window", [(1.0, None), (2.0 ** -6, None), (2.0 ** -6, 97)])
@pytest.mark.parametrize("B,T,HQ,H,D,pages,_,block,lengths,counts", ATTENTION + [
    (2, 515, 32, 8, 128, 12, "", "causal", [200, 3], None),        # several row tiles a workgroup
    (32, 64, 32, 8, 64, 3, "", "full", [4 * b for b in range(32)], None),
])
def test_outputs_are_within_the_two_parts_bound(pkg, dev, B, T, HQ, H, D, pages, _, block, lengths, counts, sharp,
                                                 window):
    say("weight parts", B, T, HQ, H, D, pages, block, lengths, counts, sharp, window)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, "bf16", block, lengths, counts, 3 + B * T,
                                       sharp)
    sinks = 5 if window else 0
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), counts=ints(counts, dev), window=window,
                                 sinks=sinks, block=block if masks is None else masks.to(dev), weight_parts=2)
    torch.cuda.synchronize()
    assert outside(cache, q, lengths, counts, block, masks, window, sinks, out, lse, "bf16", 2) == 0


@pytest.mark.parametrize("T", [1, 20, 600])
def test_values_that_cancel(pkg, dev, T):
    """Slots in pairs of equal keys and nearly opposite values: what is left is far below what the weights moved."""
    say("cancelling values", T)
    HQ, H, D, n = 8, 2, 128, 640
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randint(-15, 16, (1, n // 2, H, D), generator=g).float() / 8 for _ in "kv")
    v = torch.stack([v, -v + (torch.rand(v.shape, generator=g) < 0.02) / 8.0], 2).view(1, n, H, D)
    k = (k[:, :, None] + torch.randint(-1, 2, (1, n // 2, 2, H, D), generator=g) / 8).view(1, n, H, D)
    cache = pkg.KV8Cache.allocate(1, n + T, H, D, dev)
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = (torch.randn(1, T, HQ, D, generator=g) * 0.05).to(torch.bfloat16)
    for parts in (1, 2):
        out, lse = pkg.kv8_attention(q.to(dev), cache, ints([n], dev), block="none", weight_parts=parts)
        torch.cuda.synchronize()
        assert outside(cache, q, [n], None, "none", None, None, 0, out, lse, "bf16", parts) == 0


@pytest.mark.parametrize("T", [1, 8, 64])
def test_two_parts_are_not_one(pkg, dev, T):
    """Six slots whose values leave little: one part's rounding (2^-12 of a weight on average, over the root of six
    slots) is several times what the bound of two parts allows."""
    say("few slots", T)
    HQ, H, D, n = 8, 1, 128, 6
    g = torch.Generator().manual_seed(T)
    k = torch.randint(-15, 16, (1, n, H, D), generator=g).float() / 8
    v = torch.randint(-15, 16, (1, n // 2, H, D), generator=g).float() / 8
    v = torch.cat([v, -v], 1)
    cache = pkg.KV8Cache.allocate(1, n + T, H, D, dev)
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = (torch.randn(1, T, HQ, D, generator=g) * 0.05).to(torch.bfloat16)
    bad = {}
    for parts in (1, 2):
        out, lse = pkg.kv8_attention(q.to(dev), cache, ints([n], dev), block="none", weight_parts=parts)
        torch.cuda.synchronize()
        assert outside(cache, q, [n], None, "none", None, None, 0, out, lse, "bf16", parts) == 0
        bad[parts] = outside(cache, q, [n], None, "none", None, None, 0, out, lse, "bf16", 2)
    assert bad[2] == 0 and bad[1] > 0


def test_fp16_outputs_have_two_parts_as_it_is(pkg, dev):
    say("fp16 parts")
    lengths = [700, 3]
    cache, q, _ = attention_inputs(pkg, dev, 2, 5, 12, 4, 128, 12, "f16", "causal", lengths, None, 9)
    one, two = (pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), weight_parts=p) for p in (1, 2))
    torch.cuda.synchronize()
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    # and rows that are not held, and trees with positions, as ever
    cache, q, masks = attention_inputs(pkg, dev, 2, 9, 8, 2, 64, 4, "bf16", "mask", [120, 60], None, 4)
    K = torch.full((2, 1, 2, 64), float("nan"), device=dev)
    pkg.kv8_append(cache, K, K, ints([100, 3], dev))
    at = (torch.tensor([[120], [60]]) + torch.arange(9) // 2).int().to(dev)
    kw = dict(block=masks.to(dev), window=25, sinks=2, positions=at)
    one, two = (pkg.kv8_attention(q.to(dev), cache, ints([120, 60], dev), weight_parts=p, **kw) for p in (1, 2))
    torch.cuda.synchronize()
    assert torch.equal(one[1].isnan(), two[1].isnan()) and torch.equal(one[0].isnan(), two[0].isnan())
    f = ~one[1].isnan()
    assert one[1].isnan().any() and f.any()
    assert torch.all((one[1] - two[1])[f].abs() <= 2.0 ** -18 * (1 + two[1][f].abs()))
    assert np.array_equal(contents(cache)[0][0, 0, 100], np.full(64, np.nan), equal_nan=True)


@pytest.mark.parametrize("block,window,sinks", [("causal", None, 0), ("mask", 100, 70), ("none", 130, 64)])
@pytest.mark.parametrize("T,D", [(4, 128), (8, 64), (16, 128), (32, 64), (64, 128)])
def test_two_parts_over_pages_of_all_kinds(pkg, dev, T, D, block, window, sinks):
    """One, two, four and eight row tiles a workgroup, over pages that the table does not name, rows that are not
    held and partial pages; in the queries' place, too."""
    say("two parts, pages of all kinds", T, D, block, window, sinks)
    B, H, G, pages = 32, 8, 4, 9
    lengths = [(37 * b + 5) % (64 * pages - T) if b != 3 else 0 for b in range(B)]
    counts = [T if b % 4 else (11 * b) % (T + 1) for b in range(B)]
    cache, q, masks = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, "bf16", block, lengths, counts, T + D)
    ends = [n if block == "none" else n + c for n, c in zip(lengths, counts)]
    for b in range(0, B, 3):                                       # a row of one head that is not held
        slot = (29 * b) % max(1, ends[b])
        at = 128 * D + 8 * (slot // 32 % 2) + 4 + slot % 32 // 8
        cache.data[cache.block_table[b, slot // 64].item(), b % H, at] |= 1 << slot % 8
    K, V = contents(cache)
    named = np.ones((B, 64 * pages), bool)
    for b in range(1, B, 2):
        p = (5 * b) % pages
        cache.block_table[b, p] = (-1, 10 ** 9, cache.data.shape[0])[b % 3]
        named[b, 64 * p:64 * p + 64] = False
    for b, n in enumerate(ends):                                   # what was spoiled is not there
        K[b, :, n:], V[b, :, n:] = 0, 0
    kw = dict(counts=ints(counts, dev), window=window, sinks=sinks, block=block if masks is None else masks.to(dev),
              weight_parts=2)
    n, qd = ints(lengths, dev), q.to(dev)
    out, lse = pkg.kv8_attention(qd, cache, n, **kw)
    torch.cuda.synchronize()
    check(q, K, V, named, lengths, counts, block, masks, window, sinks, out, lse, "bf16", D ** -0.5)
    there, again = pkg.kv8_attention(qd, cache, n, out=qd, **kw)
    torch.cuda.synchronize()
    assert there is qd and same(qd, out) and same(again, lse)
