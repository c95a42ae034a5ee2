"""GPU tests of the 4-bit cache's calls at the edges of what they take."""

import pytest
import torch

from test_gpu_kv4 import attention_inputs, ints, say

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
