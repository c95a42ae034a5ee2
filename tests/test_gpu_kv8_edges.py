"""GPU tests of the 8-bit cache's edges: strides, streams, graphs, pages that are none, and refusals."""

import pytest
import torch

from test_gpu_kv8 import (attention_inputs, check_attention, contents, ints, random_cache, same, say, tables,
                          unpacked)
from oracle import kv8 as O

pytestmark = pytest.mark.gpu


def test_strides_given_outputs_and_other_streams(pkg, dev):
    say("strides")
    B, T, HQ, H, D = 2, 5, 4, 2, 64
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, 3, "bf16", "causal", [100, 30], None, 9)
    wide = torch.zeros(B, HQ, T, 3 * D, dtype=q.dtype)
    wide[..., D:2 * D] = q.transpose(1, 2)
    qv = wide.to(dev)[..., D:2 * D].transpose(1, 2)
    out = torch.full((B, HQ, T, 2 * D), 7.0, dtype=q.dtype, device=dev)
    lse = torch.empty(B, T, HQ, device=dev)
    lengths = ints([100, 30], dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        o, l = pkg.kv8_attention(qv, cache, lengths, out=out[..., :D].transpose(1, 2), lse=lse, window=70, sinks=2)
    side.synchronize()
    assert o.data_ptr() == out.data_ptr() and l is lse and torch.all(out[..., D:] == 7)
    check_attention(cache, q, "bf16", "causal", [100, 30], None, None, D ** -0.5, o, l, 70, 2)
    # keys, values and queries as parts of one projection's output
    rows = torch.randn(B, T, HQ + 2 * H, D, device=dev).to(torch.bfloat16)
    a, b = (random_cache(pkg, dev, B, H, D, 3, seed=1) for _ in "ab")
    rotary = pkg.RotaryTable(*tables(200, D, dev))
    pq, pk, pv = rows.split((HQ, H, H), 2)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        one = pkg.kv8_append(a, pk, pv, lengths, rotary=rotary, q=pq)
    side.synchronize()
    two = pkg.kv8_append(b, pk.contiguous(), pv.contiguous(), lengths, rotary=rotary, q=pq.contiguous())
    torch.cuda.synchronize()
    assert torch.equal(one, two) and torch.equal(a.data, b.data)


def test_one_tree_and_one_row_of_pages_for_all_sequences(pkg, dev):
    say("shared rows")
    B, T, HQ, H, D = 3, 6, 4, 2, 64
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, 4, "bf16", "mask", [100] * 3, None, 2)
    row = cache.block_table[:1].clone()
    shared = pkg.KV8Cache(cache.data, row.expand(B, 4), D)
    own = pkg.KV8Cache(cache.data, row.repeat(B, 1), D)
    tree = masks[:1].to(dev)
    got = pkg.kv8_attention(q.to(dev), shared, ints([100] * 3, dev), block=tree.expand(B, T))
    want = pkg.kv8_attention(q.to(dev), own, ints([100] * 3, dev), block=tree.repeat(B, 1))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k = [pkg.kv8_read(c, ints([3] * 3, dev), 90) for c in (shared, own)]
    assert all(torch.equal(x, y) for x, y in zip(*k))


def test_lengths_counts_and_pages_out_of_range(pkg, dev):
    """Clamped lengths and counts; entries that name no page hold nothing and take nothing."""
    say("out of range")
    B, T, HQ, H, D = 4, 3, 4, 2, 64
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, 3, "bf16", "full", [150, 192, 0, 60], None, 12)
    cache.block_table[0, 1], cache.block_table[3, 0] = -5, 10 ** 6
    before = cache.data.clone()
    wild = ints([150, 10 ** 9, -7, 60], dev)
    counts = ints([10 ** 6, 2, -1, 3], dev)
    out, lse = pkg.kv8_attention(q.to(dev), cache, wild, block="full", counts=counts)
    torch.cuda.synchronize()
    K, V = contents_of_named(cache)
    see = {0: list(range(64)) + list(range(128, 153)), 1: list(range(192)), 2: [], 3: []}
    for b, slots in see.items():
        for t in range(T):
            if not slots or t >= [3, 2, 0, 3][b]:
                assert torch.all(lse[b, t] == -float("inf")) and not out[b, t].any()
                continue
            for hq in range(HQ):
                k, v = (torch.tensor(x[b, hq // 2][slots]) for x in (K, V))
                row = q[b, t, hq].double() * D ** -0.5
                x, err = k @ row, (k.abs() @ row.abs()).max().item() * 2.0 ** -16
                p, rl = torch.softmax(x, 0), torch.logsumexp(x, 0).item()
                assert abs(lse[b, t, hq].item() - rl) <= err + 2.0 ** -20 * (1 + abs(rl))
                off = (p @ v.abs()) * (2.0 ** -11 + 2.0 ** -16 + 2 * err + 2.0 ** -19)    # an f16 weight
                want = p @ v                               # and half a step of bf16
                assert torch.all((out[b, t, hq].double().cpu() - want).abs() <= off + (want.abs() + off) * 2.0 ** -8)
    # slots past the table's, entries of no page: nothing is written anywhere
    kv = torch.randn(B, T, H, D, device=dev).to(torch.bfloat16)
    pkg.kv8_append(cache, kv, kv, ints([70, 2 ** 31 - 1, 191, 10], dev), counts=ints([3, 3, 0, 3], dev))
    torch.cuda.synchronize()
    assert torch.equal(cache.data, before)
    k, v = pkg.kv8_read(cache, ints([62, 190, 2 ** 31 - 1, 0], dev), 5)
    torch.cuda.synchronize()
    assert k[0, :2].any() and not k[0, 2:].any() and not v[0, 2:].any()
    assert k[1, :2].any() and not k[1, 2:].any() and not k[2:].any() and not v[2:].any()


def contents_of_named(cache):
    table = cache.block_table.clamp(0, cache.data.shape[0] - 1)
    kc, ke, vc, ve, bad = O.unpack(cache.data.cpu().numpy(), table.cpu().numpy(), cache.head_dim)
    return O.values(kc, ke, bad), O.values(vc, ve, bad)


@pytest.mark.parametrize("pages,columns", [(0, 3), (3, 0)])
def test_caches_of_no_pages_and_tables_of_no_columns(pkg, dev, pages, columns):
    say("nothing", pages, columns)
    cache = pkg.KV8Cache(torch.zeros(pages, 2, 8320, dtype=torch.uint8, device=dev),
                         torch.zeros(2, columns, dtype=torch.int32, device=dev), 64)
    n = ints([100, 0], dev)
    q, kv = (torch.randn(2, 3, h, 64, device=dev).to(torch.bfloat16) for h in (4, 2))
    rotary = pkg.RotaryTable(*tables(200, 64, dev))
    turned = pkg.kv8_append(cache, kv, kv, n, rotary=rotary, q=q)
    k, v = pkg.kv8_read(cache, n, 3)
    out, lse = pkg.kv8_attention(q, cache, n)
    o2, l2 = pkg.kv8_attention(q, cache, n, window=5, sinks=70)
    torch.cuda.synchronize()
    assert not k.any() and not v.any() and not cache.data.any()
    for o, l in ((out, lse), (o2, l2)):
        assert not o.any() and torch.all(l == -float("inf"))
    # queries are rotated all the same; positions follow the length that the table can hold
    at = [min(x, 64 * columns) for x in (100, 0)]
    c, s = (t.cpu().numpy() for t in tables(200, 64, dev))
    import numpy as np
    want = np.stack([O.rotate(q.float().cpu().numpy()[:, :, h], c, s, np.array(at)[:, None] + np.arange(3), False)
                     for h in range(4)], 2)
    assert same(turned.cpu(), torch.tensor(want).to(torch.bfloat16))


def test_a_block_of_no_rows(pkg, dev):
    say("empty block")
    B, HQ, H, D = 3, 4, 2, 64
    cache = random_cache(pkg, dev, B, H, D, 5, seed=1)
    before, n = cache.data.clone(), ints([0, 300, 77], dev)
    q, kv = (torch.zeros(B, 0, h, D, dtype=torch.bfloat16, device=dev) for h in (HQ, H))
    rotary = pkg.RotaryTable(*tables(20, D, dev))
    turned = pkg.kv8_append(cache, kv, kv, n, rotary=rotary, q=q)
    k, v = pkg.kv8_read(cache, n, 0)
    out, lse = pkg.kv8_attention(q, cache, n)
    torch.cuda.synchronize()
    assert k.shape == v.shape == (B, 0, H, D) and out.shape == turned.shape == q.shape and lse.shape == (B, 0, HQ)
    assert torch.equal(cache.data, before)


def test_repeated_calls_are_bit_identical(pkg, dev):
    say("repeat")
    for T in (1, 16, 200):
        cache, q, _ = attention_inputs(pkg, dev, 3, T, 8, 2, 128, 25, "bf16", "causal", [1200, 700, 3], None, 31)
        lengths, qd = ints([1200, 700, 3], dev), q.to(dev)
        first = pkg.kv8_attention(qd, cache, lengths)
        for _ in range(5):
            o, l = pkg.kv8_attention(qd, cache, lengths)
            assert torch.equal(o, first[0]) and torch.equal(l, first[1])


def test_calls_replay_in_a_graph(pkg, dev):
    """Append with rotation, attention whole and through a window, captured once and replayed on new inputs."""
    say("graph")
    B, T, HQ, H, D, S = 2, 4, 8, 2, 128, 512
    caches = [pkg.KV8Cache.allocate(B, S, H, D, dev) for _ in range(2)]
    rotary = pkg.RotaryTable(*tables(S, D, dev))
    g = torch.Generator(device=dev).manual_seed(4)
    q = torch.empty(B, T, HQ, D, dtype=torch.bfloat16, device=dev)
    k, v = (torch.empty(B, T, H, D, dtype=torch.bfloat16, device=dev) for _ in "kv")
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)

    def step(cache, lengths):
        turned = pkg.kv8_append(cache, k, v, lengths, rotary=rotary, q=q)
        return (turned, *pkg.kv8_attention(turned, cache, lengths),
                *pkg.kv8_attention(turned, cache, lengths, window=50, sinks=4), *pkg.kv8_read(cache, lengths, T))

    def fill():
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))

    fill()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(caches[0], lengths)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    caches[0].data.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0], lengths)
        lengths += T
    el = torch.zeros_like(lengths)
    lengths.zero_()
    for i in range(40):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        eager = step(caches[1], el)
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), i
        el = el + T
    assert torch.equal(caches[0].data, caches[1].data)


def test_graphs_of_one_cache_are_replayed_on_two_streams(pkg, dev):
    say("two graphs at once")
    cache = random_cache(pkg, dev, 2, 2, 64, 70, seed=1)
    lengths = ints([4000, 3000], dev)
    qs = [torch.empty(2, T, 8, 64, dtype=torch.bfloat16, device=dev) for T in (2, 20)]
    g = torch.Generator(device=dev).manual_seed(7)
    streams = [torch.cuda.Stream(dev) for _ in qs]
    streams[0].wait_stream(torch.cuda.current_stream(dev))
    graphs = []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            got = pkg.kv8_attention(q, cache, lengths, block="none")
        graphs.append((graph, got))
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
            for x, y in zip(got, pkg.kv8_attention(q, cache, lengths, block="none")):
                assert torch.equal(x, y)


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
    far = pkg.KV8Cache(data, small.block_table + first, D)
    rotary = pkg.RotaryTable(*tables(400, D, dev))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(B, T, H, D, generator=g).to(torch.bfloat16).to(dev) for _ in "kv")
    n, made = ints([300, 333], dev), []
    for cache in (small, far):
        turned = pkg.kv8_append(cache, k, v, n, rotary=rotary, q=q.to(dev))
        made.append((turned, *pkg.kv8_attention(turned, cache, n), *pkg.kv8_attention(turned, cache, n, window=90),
                     *pkg.kv8_read(cache, ints([200, 200], dev), 130)))
    torch.cuda.synchronize()
    for x, y in zip(*made):                                    # what is read past the rows is NaN here
        assert same(x, y)
    assert torch.equal(far.data[first:], small.data)


def test_a_text_through_the_cache_in_blocks(pkg, dev):
    """Rows appended in uneven blocks, some rejected, attended as they come: as one pass over what the cache holds."""
    say("together")
    B, HQ, H, D, S = 2, 8, 2, 128, 400
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(B, S, h, D, generator=g).to(torch.bfloat16) for h in (HQ, H, H))
    cos, sin = tables(S, D, dev)
    rotary = pkg.RotaryTable(cos, sin)
    cache = pkg.KV8Cache.allocate(B, S, H, D, dev)
    lengths = ints([0, 0], dev)
    at = 0
    for T, stay in ((150, 150), (1, 1), (16, 5), (16, 16), (7, 1), (64, 60), (33, 33), (1, 1), (16, 9)):
        block = [x[:, at:at + T].to(dev) for x in (q, k, v)]
        turned = pkg.kv8_append(cache, block[1], block[2], lengths, rotary=rotary, q=block[0])
        for window, sinks in ((None, 0), (40, 4)):
            out, lse = pkg.kv8_attention(turned, cache, lengths, window=window, sinks=sinks)
            torch.cuda.synchronize()
            check_attention(cache, turned.cpu(), "bf16", "causal", [at] * B, None, None, D ** -0.5, out, lse, window,
                            sinks)
        at += stay
        lengths = lengths + stay
    # what the cache holds is near what went in: e4m3 by half a step of 2^-4, twice where a block's
    # exponent rose, 2^-10 of the block's 448-fold below its normal numbers
    kr, vr = pkg.kv8_read(cache, ints([0, 0], dev), at, dtype=torch.float32)
    torch.cuda.synchronize()
    c, s = cos.cpu()[:at, None], sin.cpu()[:at, None]
    a, b = k[:, :at].float().chunk(2, -1)
    kt = torch.cat((a * c - b * s, b * c + a * s), -1)
    for got, want in ((kr.cpu(), kt), (vr.cpu(), v[:, :at].float())):
        assert torch.all((got - want).abs() <= want.abs() * 2.0 ** -3 + want.abs().max() * 2.0 ** -15)


def test_refusals(pkg, dev):
    cache = pkg.KV8Cache.allocate(2, 100, 2, 64, dev)
    assert cache.slots == 128 and cache.data.shape == (4, 2, 8320)
    bf = torch.bfloat16
    q = torch.zeros(2, 3, 4, 64, dtype=bf, device=dev)
    kv = torch.zeros(2, 3, 2, 64, dtype=bf, device=dev)
    n = ints([0, 0], dev)
    rotary = pkg.RotaryTable(*tables(200, 64, dev))
    with pytest.raises(ValueError, match="head_dim must be one of"):
        pkg.KV8Cache.allocate(1, 64, 1, 80, dev)
    with pytest.raises(ValueError, match="no CPU fallback"):
        pkg.kv8_append(cache, kv.cpu(), kv, n)
    with pytest.raises(ValueError, match="no CPU fallback"):
        pkg.RotaryTable(torch.zeros(4, 32), torch.zeros(4, 32))
    with pytest.raises(ValueError, match="one shape and dtype"):
        pkg.kv8_append(cache, kv, kv.float(), n)
    with pytest.raises(ValueError, match="lengths must be int32"):
        pkg.kv8_append(cache, kv, kv, n.long())
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        odd = torch.zeros(2, 3, 2, 67, dtype=bf, device=dev)[..., :64]
        pkg.kv8_append(cache, odd, odd, n)
    with pytest.raises(RuntimeError, match="rotary rows"):
        t = torch.zeros(200, 33, device=dev)[:, :32]
        pkg.kv8_append(cache, kv, kv, n, rotary=pkg.RotaryTable(t, t))
    with pytest.raises(ValueError, match="q must be"):
        pkg.kv8_append(cache, kv, kv, n, rotary=rotary, q=q[:, :, :3])
    with pytest.raises(TypeError, match="q dtype"):
        pkg.kv8_attention(q.float(), cache, n)
    with pytest.raises(ValueError, match="do not divide"):
        pkg.kv8_attention(q[:, :, :3], cache, n)
    with pytest.raises(RuntimeError, match="holds 64 slots"):
        pkg.kv8_attention(torch.zeros(2, 65, 4, 64, dtype=bf, device=dev), cache, n,
                          block=torch.zeros(2, 65, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="scale must be finite"):
        pkg.kv8_attention(q, cache, n, scale=float("nan"))
    with pytest.raises(ValueError, match="sinks are for a window"):
        pkg.kv8_attention(q, cache, n, sinks=4)
    with pytest.raises(TypeError, match="bits a value"):
        pkg.kv8_attention(q, pkg.KV4Cache.allocate(2, 100, 2, 64, dev), n)
    with pytest.raises(TypeError, match="bits a value"):
        pkg.kv4_attention(q, cache, n)
    # nothing was written
    assert not cache.data.any() and not unpacked(cache)[4].any() and not contents(cache)[0].any()
