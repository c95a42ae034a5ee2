"""GPU tests of the 4-bit cache's calls at the edges of what they take."""

import numpy as np
import pytest
import torch

from oracle import kv4 as O
from test_gpu_kv4 import DT, attention_inputs, check_attention, contents, ints, say

pytestmark = pytest.mark.gpu


def test_one_tree_and_one_row_of_pages_for_all_sequences(pkg, dev):
    """Expanded masks and tables: as their copies."""
    say("expanded mask and table")
    B, T, HQ, H, D = 5, 7, 4, 2, 64
    cache, q, _ = attention_inputs(pkg, dev, 1, T, HQ, H, D, 3, "bf16", "full", [130], None, 12)
    qd = q.expand(B, T, HQ, D).contiguous().to(dev)
    table = cache.block_table.expand(B, -1)
    mask = torch.tensor([(1 << t) | (t and 1) for t in range(T)], device=dev)[None]
    n = ints([130, 64, 5, 0, 100], dev)
    made = []
    for tab, m in ((table, mask.expand(B, T)), (table.contiguous(), mask.repeat(B, 1))):
        c = pkg.KV4Cache(cache.data, tab, D)
        out, lse = pkg.kv4_attention(qd, c, n, block=m)
        w = pkg.kv4_weights(qd, c, n, lse, torch.zeros(B, H, c.slots, device=dev), block=m)
        made.append((out, lse, w, *pkg.kv4_read(c, n, 9)))
    torch.cuda.synchronize()
    for x, y in zip(*made):                                # as bits: the slots past 136 hold NaN
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    assert torch.isfinite(made[0][1]).all()


def two_blocks(pkg, dev):
    """A cache whose rows are split among workgroups, and queries of two block lengths to be filled."""
    B, HQ, H, D = 2, 8, 2, 128
    cache, _, _ = attention_inputs(pkg, dev, B, 1, HQ, H, D, 90, "bf16", "none", [5500, 4000], None, 40)
    return cache, ints([5500, 4000], dev), [torch.zeros(B, T, HQ, D, dtype=torch.bfloat16, device=dev) for T in (17, 2)]


def capture(stream, step):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    return graph, out


@pytest.mark.parametrize("kept", [False, True])
def test_graphs_are_replayed_in_any_order(pkg, dev, kept):
    """Two graphs captured on one stream, the second replayed first, larger eager calls there in between."""
    say("two graphs", kept)
    cache, lengths, qs = two_blocks(pkg, dev)
    spare = pkg.KV4Cache(cache.data.clone(), cache.block_table, 128)
    g = torch.Generator(device=dev).manual_seed(6)
    wide = torch.randn(2, 64, 8, 128, generator=g, device=dev).to(torch.bfloat16)
    w = torch.rand(2, 2, cache.slots, generator=g, device=dev)
    ws = pkg.ops.new_workspace(dev, 1 << 25) if kept else None

    def step(q, given=None):
        return (*pkg.kv4_attention(q, cache, lengths, block="none", workspace=given),
                *pkg.kv4_evict(spare, lengths, w, 3000 + q.shape[1], 8, workspace=given))

    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    graphs = [capture(stream, lambda: step(q, ws)) for q in qs]
    for i in (1, 0, 1, 1, 0, 0, 1):
        qs[i].copy_(torch.randn(qs[i].shape, generator=g, device=dev))
        spare.data.copy_(cache.data)
        stream.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(stream):
            pkg.kv4_attention(wide, cache, lengths, block="none")
            graphs[i][0].replay()
        torch.cuda.synchronize()
        moved = spare.data.clone()
        spare.data.copy_(cache.data)
        for x, y in zip((*graphs[i][1], moved), (*step(qs[i]), spare.data)):
            assert torch.equal(x, y), i


def test_graphs_of_one_cache_are_replayed_on_two_streams(pkg, dev):
    say("two graphs at once")
    cache, lengths, qs = two_blocks(pkg, dev)
    g = torch.Generator(device=dev).manual_seed(7)
    streams = [torch.cuda.Stream(dev) for _ in qs]
    graphs = [capture(streams[0], lambda: pkg.kv4_attention(q, cache, lengths, block="none")) for q in qs]
    for _ in range(5):
        for q in qs:
            q.copy_(torch.randn(q.shape, generator=g, device=dev))
        torch.cuda.synchronize()
        for _ in range(4):
            for (graph, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for q, (_, got) in zip(qs, graphs):
            for x, y in zip(got, pkg.kv4_attention(q, cache, lengths, block="none")):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,T,block", [("bf16", 3, "causal"), ("f16", 9, "full"), ("bf16", 40, "causal")])
def test_rows_of_nan_and_infinite_queries(pkg, dev, dtype, T, block):
    """Their out and lse are NaN, and the weights of the slots that they see; other rows are as ever."""
    say("nan rows", dtype, T, block)
    B, HQ, H, D, lengths, counts = 3, 4, 2, 64, [130, 700, 0], [T, T, T - 1]
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, 12, dtype, block, lengths, counts, 17)
    bad = torch.zeros(B, T, HQ, dtype=torch.bool)
    for (b, t, hq), x in {(0, 0, 1): "nan", (0, T - 2, 0): "inf", (1, 1, 3): "-inf", (1, T - 1, 3): "nan",
                          (2, 1, 0): "nan"}.items():
        q[b, t, hq, 7 * hq + 2] = float(x)
        bad[b, t, hq] = True
    q[2, T - 1] = float("nan")                             # no valid row
    n, c = ints(lengths, dev), ints(counts, dev)
    out, lse = pkg.kv4_attention(q.to(dev), cache, n, block=block, counts=c)
    torch.cuda.synchronize()
    assert torch.equal(lse.cpu().isnan(), bad)
    assert torch.equal(out.cpu().isnan(), bad[..., None].expand_as(out))
    # the other rows, as without the bad ones
    clean = torch.where(bad[..., None] | q.isnan(), torch.zeros_like(q), q)
    o, l = out.cpu(), lse.cpu()
    co, cl = (x.cpu() for x in pkg.kv4_attention(clean.to(dev), cache, n, block=block, counts=c))
    o[bad], l[bad] = co[bad], cl[bad]
    check_attention(cache, clean, dtype, block, lengths, counts, None, D ** -0.5, o, l)

    w = torch.rand(B, H, cache.slots, generator=torch.Generator().manual_seed(2))
    K, _ = contents(cache)
    for accepted in (counts, [1, 1, 1]):
        got = pkg.kv4_weights(q.to(dev), cache, n, lse, w.to(dev), ints(accepted, dev), block=block, counts=c)
        with np.errstate(invalid="ignore"):
            ref, added, mass = O.weights(q.double().numpy(), K, lengths, counts, accepted, block, D ** -0.5,
                                         lse.double().cpu().numpy(), w.double().numpy())
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert np.isnan(ref).any() and not np.isnan(ref).all()
        f = ~np.isnan(ref)
        err = np.abs(clean.double().numpy()).sum(-1).max() * 6 * 2.0 ** -16      # keys are 6 at most
        assert np.all(np.abs(got - ref)[f] <= (added * (err + 2.0 ** -18) + ref * 2.0 ** -20)[f])


def test_rows_of_minus_infinite_scores_are_empty(pkg, dev):
    """Every score -inf: nothing is seen, though slots are; a score of -inf beside others weighs nothing."""
    say("-inf scores")
    D = 64
    cache = pkg.KV4Cache.allocate(1, 128, 1, D, dev)
    k = torch.ones(1, 100, 1, D, device=dev)
    k[0, :50, 0, 3] = 0.0                                  # with a query of -inf there: NaN
    pkg.kv4_append(cache, k, k, ints([0], dev))
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16, device=dev)
    q[0, 0, 0, 5] = float("-inf")
    q[0, 1, 0, 3] = float("-inf")
    out, lse = pkg.kv4_attention(q, cache, ints([100], dev), block="none")
    torch.cuda.synchronize()
    assert lse[0, 0, 0] == float("-inf") and not out[0, 0].any()
    assert lse[0, 1, 0].isnan() and out[0, 1].isnan().all()


@pytest.mark.parametrize("n,pages,keep,recent,gone", [
    (500, 8, 200, 30, [1, 6]),                             # below and above the budget
    (500, 8, 200, 30, [3]),                                # the budget ends inside a page that is none
    (500, 8, 200, 200, [0, 2]),                            # fewer places than recent slots
    (500, 8, 128, 100, [0, 1, 5]),                         # no place at all
    (500, 8, 200, 150, [7, 6]),                            # the recent slots are in no page
    (500, 8, 200, 0, list(range(8))),                      # nothing anywhere
    (20000, 320, 9000, 500, [0, 17, 140, 141, 200, 311]),  # several walks of the selection
    (500, 8, 600, 10, [1, 2]),                             # a budget that is kept
])
def test_evict_beside_entries_that_name_no_page(pkg, dev, n, pages, keep, recent, gone):
    """No slot there stays, moves or is moved into, and what is said of every place is what it holds."""
    say("evict no page", n, pages, keep, recent, gone)
    B, H, D = 2, 2, 64
    g = torch.Generator().manual_seed(n + keep + len(gone))
    data = torch.randint(0, 256, (B * pages, H, O.page_bytes(D)), generator=g, dtype=torch.uint8)
    data[..., 32 * D:34 * D] = torch.randint(100, 140, (B * pages, H, 2 * D), generator=g, dtype=torch.uint8)
    data[..., 66 * D:] = (torch.rand(B * pages, H, 64, generator=g) + 0.1).to(torch.bfloat16).view(torch.uint8)
    table = torch.randperm(B * pages, generator=g).view(B, pages).int()
    for i, p in enumerate(gone):
        table[0, p] = -1 if i % 2 else 10 ** 6
    cache = pkg.KV4Cache(data.to(dev), table.to(dev), D)
    w = torch.randint(0, 50, (B, H, cache.slots), generator=g).float()
    lengths = ints([n, n], dev)
    k0, v0 = pkg.kv4_read(cache, ints([0, 0], dev), n, dtype=torch.float32)
    nl, nw, source = pkg.kv4_evict(cache, lengths, w.to(dev), keep, recent)
    k1, v1 = pkg.kv4_read(cache, ints([0, 0], dev), min(n, keep), dtype=torch.float32)
    torch.cuda.synchronize()
    m = min(n, keep)
    assert nl.tolist() == [m, m]
    for b in range(B):
        named = np.array([0 <= int(table[b, j // 64]) < B * pages for j in range(n)])
        for h in range(H):
            ref = O.evict(w[b, h, :n].double().numpy(), n, keep, recent, named)
            assert np.array_equal(source[b, h].cpu().numpy(), ref), (b, h)
            src = torch.tensor(ref[:m])
            assert torch.equal(nw[b, h, :m].cpu(), w[b, h][src]) and not nw[b, h, m:].any()
            for x, y in ((k0, k1), (v0, v1)):
                assert torch.equal(x[b, src.to(dev), h], y[b, :, h])


def test_cache_whose_table_has_no_column(pkg, dev):
    say("no column")
    cache = pkg.KV4Cache(torch.zeros(3, 2, 4352, dtype=torch.uint8, device=dev),
                         torch.zeros(2, 0, dtype=torch.int32, device=dev), 64)
    n = ints([5, 0], dev)
    q, kv = (torch.randn(2, 3, h, 64, device=dev).to(torch.bfloat16) for h in (4, 2))
    w = torch.zeros(2, 2, 0, device=dev)
    pkg.kv4_append(cache, kv, kv, n)
    k, v = pkg.kv4_read(cache, n, 3)
    out, lse = pkg.kv4_attention(q, cache, n)
    nw = pkg.kv4_weights(q, cache, n, lse, w)
    nl, ew, source = pkg.kv4_evict(cache, n, w, 4, 2)
    torch.cuda.synchronize()
    assert not k.any() and not v.any() and not out.any() and torch.all(lse == float("-inf"))
    assert nw.shape == ew.shape == (2, 2, 0)
    assert nl.tolist() == [0, 0] and torch.all(source == -1) and not cache.data.any()


@pytest.mark.parametrize("pages", [5, 0])
def test_a_block_of_no_rows_through_every_call(pkg, dev, pages):
    """Nothing is written or attended to; the weights of the context stay, those past it go."""
    say("empty block", pages)
    B, HQ, H, D = 3, 4, 2, 64
    data = torch.randint(0, 256, (B * pages, H, O.page_bytes(D)), dtype=torch.uint8, device=dev)
    cache = pkg.KV4Cache(data, torch.arange(B * 5, dtype=torch.int32, device=dev).view(B, 5), D)
    before, n = data.clone(), ints([0, 300, 77], dev)
    q, kv = (torch.zeros(B, 0, h, D, dtype=torch.bfloat16, device=dev) for h in (HQ, H))
    w = torch.rand(B, H, cache.slots, device=dev)
    pkg.kv4_append(cache, kv, kv, n)
    k, v = pkg.kv4_read(cache, n, 0)
    out, lse = pkg.kv4_attention(q, cache, n)
    nw = pkg.kv4_weights(q, cache, n, lse, w)
    same = w.clone()
    assert pkg.kv4_weights(q, cache, n, lse, same, ints([0, 0, 0], dev), block="none", out=same) is same
    torch.cuda.synchronize()
    assert k.shape == v.shape == (B, 0, H, D) and out.shape == q.shape and lse.shape == (B, 0, HQ)
    j = torch.arange(cache.slots, device=dev)
    want = torch.where(j < n[:, None, None], w, torch.zeros_like(w))
    assert torch.equal(nw, want) and torch.equal(same, want) and torch.equal(data, before)


@pytest.mark.parametrize("T,n,dtype,step", [(1, 700, "bf16", 0.0), (3, 700, "bf16", 0.01), (40, 300, "bf16", 0.02),
                                            (2, 5000, "f16", 0.001)])
def test_values_up_to_what_the_cache_holds(pkg, dev, T, n, dtype, step):
    """Values of 3e38 (and infinity, held as that), under even weights and rising ones: no sum overflows."""
    say("large values", T, n, dtype, step)
    HQ, H, D = 4, 2, 64
    g = torch.Generator().manual_seed(n)
    cache = pkg.KV4Cache.allocate(1, n + T, H, D, dev)
    k = torch.zeros(1, n + T, H, D)
    k[0, :, :, 0] = (torch.arange(n + T) * 1.0)[:, None]
    v = torch.where(torch.rand(D, generator=g) < 0.5, -1.0, 1.0).expand(1, n + T, H, D) * 3e38
    v = v * (0.8 + 0.2 * torch.rand(1, n + T, H, D, generator=g))
    v[0, 5, 0, 3] = v[0, n - 1, 1, 4] = float("inf")
    pkg.kv4_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = torch.zeros(1, T, HQ, D, dtype=DT[dtype])
    q[..., 0] = 1.0
    scale = step if step else 1e-6
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints([n], dev), scale=scale)
    torch.cuda.synchronize()
    if dtype == "f16":                                     # past the type's range, as the values are
        K, V = contents(cache)
        ref = O.attention(q.double().numpy(), K, V, [n], [T], "causal", scale)[0]
        assert np.array_equal(out.cpu().numpy(), np.sign(ref) * np.inf)
    else:
        check_attention(cache, q, dtype, "causal", [n], None, None, scale, out, lse)


def test_pages_past_four_gibibytes(pkg, dev):
    """The cache's last pages, more than 2^32 bytes in: every call as on a small cache of the same pages."""
    say("far pages")
    B, T, HQ, H, D, pages = 2, 5, 8, 4, 128, 6
    small, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, "bf16", "none", [300, 333], None, 50)
    size = H * O.page_bytes(D)
    total = (1 << 32) // size + 200
    data = torch.empty(total, H, O.page_bytes(D), dtype=torch.uint8, device=dev)
    first = total - small.data.shape[0]
    assert first * size > 1 << 32
    data[first:] = small.data
    far = pkg.KV4Cache(data, small.block_table + first, D)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(B, T, H, D, generator=g).to(torch.bfloat16).to(dev) for _ in "kv")
    w = torch.rand(B, H, small.slots, generator=g).to(dev)
    n, made = ints([300, 333], dev), []
    for cache in (small, far):
        pkg.kv4_append(cache, k, v, n)
        out, lse = pkg.kv4_attention(q.to(dev), cache, n)
        nw = pkg.kv4_weights(q.to(dev), cache, n, lse, w)
        evicted = pkg.kv4_evict(cache, n + T, nw, 130, 20)
        made.append((out, lse, nw, *evicted, *pkg.kv4_read(cache, ints([0, 0], dev), 130)))
    torch.cuda.synchronize()
    for x, y in zip(*made):
        assert torch.equal(x, y)
    assert torch.equal(far.data[first:], small.data)
