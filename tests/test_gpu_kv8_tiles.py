"""GPU tests of attention over the 8-bit cache at sizes where a workgroup takes 2, 4 or 8 row tiles.

256 sequences and heads are what a workgroup for every CU needs; with four query heads to each, 8 to 64
rows a sequence are one to eight tiles of 32.  Bounds are those of test_gpu_kv8.
"""

import numpy as np
import pytest
import torch

from test_gpu_kv8 import INF, NAN, attention_inputs, contents, ints, same, say
from oracle import kv8 as O

pytestmark = pytest.mark.gpu

B, H, G = 32, 8, 4
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def check(q, K, V, named, lengths, counts, block, masks, window, sinks, out, lse, dtype, scale, steep=False):
    """Every row against 64-bit products; K, V [B, H, slots, D], NaN where a row was not finite."""
    T, D, dev = q.shape[1], q.shape[3], out.device
    slots = K.shape[2]
    most = 0.0 if steep else slots * np.nanmax(np.abs(V))
    for b in range(B):
        mask = None if masks is None else masks[b].numpy()
        see = O.visible(lengths[b], counts[b], T, slots, block, mask, window, sinks)
        see = torch.tensor(see & named[b][None]).to(dev)[:, None, None]
        k, v = (torch.tensor(x[b]).to(dev) for x in (K, V))
        lost = (see & k.isnan().any(-1)[None, :, None]).any(-1).expand(T, H, G)
        k, v = k.nan_to_num(), v.nan_to_num()
        rows = q[b].double().to(dev).view(T, H, G, D).permute(1, 0, 2, 3).reshape(H, T * G, D)

        def product(x, y):
            return torch.bmm(x, y.contiguous()).view(H, T, G, -1).permute(1, 0, 2, 3)

        x = product(rows, k.transpose(1, 2)) * scale
        mass = product(rows.abs(), k.abs().transpose(1, 2)) * abs(scale)
        mass = mass.masked_fill(~see, 0).amax(-1)
        x = x.masked_fill(~see, -INF)
        rl = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(rl > -INF, rl, torch.zeros_like(rl))[..., None])
        p = p.permute(1, 0, 2, 3).reshape(H, T * G, slots)
        ro, weight = product(p, v), product(p, v.abs())
        got, o = lse[b].double().view(T, H, G), out[b].double().view(T, H, G, D)
        assert torch.equal(got.isnan(), lost) and torch.equal(o.isnan(), lost[..., None].expand_as(o)), b
        empty = rl == -INF
        assert torch.equal(got == -INF, empty & ~lost) and not o[empty & ~lost].any(), b
        f = ~empty & ~lost
        err = mass * 2.0 ** -16
        assert torch.all((got - rl)[f].abs() <= (err + 2.0 ** -20 * (1 + rl.abs()))[f]), b
        lo, hi = O.output_range(ro.cpu().numpy(), weight.cpu().numpy(), err.cpu().numpy(), dtype, most)
        o, f = o.cpu().numpy(), f.cpu().numpy()
        assert np.all(((o >= lo) & (o <= hi))[f]), b


TILES = [(8, "bf16", 128), (16, "f16", 64), (16, "bf16", 128), (32, "bf16", 64), (31, "f16", 128), (64, "bf16", 128),
         (57, "f16", 64), (64, "f16", 128)]


@pytest.mark.parametrize("block,window,sinks", [("causal", None, 0), ("mask", 100, 70), ("full", 30, 3), ("none", 1, 0),
                                                ("causal", 130, 64)])
@pytest.mark.parametrize("T,dtype,D", TILES)
def test_tiles_over_pages_of_all_kinds(pkg, dev, T, dtype, D, block, window, sinks):
    """Pages that the table does not name, rows that are not held, partial pages and empty sequences, in one call."""
    say("tiles", T, dtype, D, block, window, sinks)
    pages = 9
    lengths = [(37 * b + 5) % (64 * pages - T) if b != 3 else 0 for b in range(B)]
    counts = [T if b % 4 else (11 * b) % (T + 1) for b in range(B)]
    cache, q, masks = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, dtype, block, lengths, counts, T + D)
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
    kw = dict(counts=ints(counts, dev), window=window, sinks=sinks, block=block if masks is None else masks.to(dev))
    n, qd = ints(lengths, dev), q.to(dev)
    out, lse = pkg.kv8_attention(qd, cache, n, **kw)
    torch.cuda.synchronize()
    check(q, K, V, named, lengths, counts, block, masks, window, sinks, out, lse, dtype, D ** -0.5)
    # in the queries' place
    there, again = pkg.kv8_attention(qd, cache, n, out=qd, **kw)
    torch.cuda.synchronize()
    assert there is qd and same(qd, out) and same(again, lse)


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("T,dtype,D", [t for t in TILES if t[0] != 31])
def test_tiles_over_blocks_of_very_different_scales(pkg, dev, T, dtype, D, up):
    """Values from 2^-60 to 2^60, block by block, where the large ones weigh nothing: the small ones count in full."""
    say("tiles and scales", T, dtype, D, up)
    n, pages = 440 - T, 7
    g = torch.Generator().manual_seed(T)
    cache = pkg.KV8Cache.allocate(B, 64 * pages, H, D, dev)
    size = (torch.arange(n + T) // 32 * 8 - 54).float()            # binary orders of a block's values
    size = size if up else -size - 1
    v = torch.randn(B, n + T, H, D, generator=g) * torch.exp2(size)[None, :, None, None]
    k = torch.zeros(B, n + T, H, D)
    k[..., 0] = -size[:, None] * 1.5                               # the larger, the less it is looked at
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0] * B, dev))
    q = torch.zeros(B, T, H * G, D, dtype=DT[dtype])
    q[..., 0] = torch.linspace(0.3, 3.0, H * G)
    # sequences of all lengths, so that wide scales begin at any page
    lengths = [n - 13 * b for b in range(B)]
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), block="full", scale=1.0)
    torch.cuda.synchronize()
    K, V = contents(cache)
    lengths = [max(m, 0) for m in lengths]                         # as the call takes them
    check(q, K, V, np.ones((B, 64 * pages), bool), lengths, [T] * B, "full", None, None, 0, out, lse, dtype, 1.0,
          steep=True)


def test_queries_of_nan_stay_in_their_rows(pkg, dev):
    say("tiles and nan")
    T, D, pages = 64, 64, 4
    lengths, counts = [64 * pages - T - 3 * b for b in range(B)], [T] * B
    cache, q, _ = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, "bf16", "causal", lengths, counts, 2)
    clean, n = q.clone(), ints(lengths, dev)
    bad = torch.zeros(B, T, H * G, dtype=torch.bool)
    bad[::5, 7::16, 3::11] = True
    q[bad] = NAN
    out, lse = pkg.kv8_attention(q.to(dev), cache, n)
    want, rl = pkg.kv8_attention(clean.to(dev), cache, n)
    torch.cuda.synchronize()
    bad = bad.to(dev)
    assert torch.equal(lse.isnan(), bad) and torch.equal(out.isnan(), bad[..., None].expand_as(out))
    out[bad], lse[bad] = want[bad], rl[bad]
    K, V = contents(cache)
    for b, m in enumerate(lengths):
        K[b, :, m + T:], V[b, :, m + T:] = 0, 0
    check(clean, K, V, np.ones((B, 64 * pages), bool), lengths, counts, "causal", None, None, 0, out, lse, "bf16",
          D ** -0.5)


@pytest.mark.parametrize("T,D,window", [(8, 128, None), (16, 128, None), (32, 64, 100), (64, 128, None)])
def test_tiles_replay_in_a_graph(pkg, dev, T, D, window):
    """Captured once and replayed on new queries and lengths, twice each, with eager calls between: the same bits."""
    say("tiles in a graph", T, D, window)
    pages = 8
    lengths = [(37 * b + 5) % (64 * pages - T) for b in range(B)]
    cache, q, _ = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, "bf16", "none", [64 * pages] * B, None, T)
    n, qd = ints(lengths, dev), q.to(dev)
    kw = dict(block="none", window=window, sinks=3 if window else 0)
    pkg.kv8_attention(qd, cache, n, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = pkg.kv8_attention(qd, cache, n, **kw)
    g = torch.Generator(device=dev).manual_seed(T)
    for i in range(4):
        qd.copy_(torch.randn(qd.shape, generator=g, device=dev))
        n.copy_(torch.roll(n, 1))
        eager = pkg.kv8_attention(qd, cache, n, **kw)
        for _ in range(2):
            for x in captured:
                x.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(captured, eager):
                assert torch.equal(x, y), i
