"""GPU tests of windows over trees: a row's window goes by its position, as decoding its branch alone would.

Bounds are those of test_gpu_kv8 (oracle.kv8.output_range).
"""

import numpy as np
import pytest
import torch

from oracle import kv8 as O
from test_gpu_kv8 import (INF, append_inputs, attention_inputs, check_append, contents, ints, random_cache, say,
                          tables, unpacked)

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def tree(T, rng, wide=0.3):
    """Bits and depths of a random tree of T rows, parents before children."""
    bits, depth = [], []
    for t in range(T):
        up = -1 if t == 0 or rng.random() < wide * (t < 4) else int(rng.integers(max(0, t - 6), t))
        bits.append((bits[up] if up >= 0 else 0) | 1 << t)
        depth.append(depth[up] + 1 if up >= 0 else 0)
    return [x - (1 << 64) if x >= 1 << 63 else x for x in bits], depth


def trees(B, T, seed, lengths):
    rng = np.random.default_rng(seed)
    made = [tree(T, rng) for _ in range(B)]
    masks = torch.tensor([m for m, _ in made], dtype=torch.int64)
    return masks, torch.tensor([[n + d for d in ds] for n, (_, ds) in zip(lengths, made)], dtype=torch.int32)


def check(cache, q, masks, positions, lengths, counts, window, sinks, out, lse, dtype):
    """Every row against 64-bit products over the slots that it sees; what lies behind the blocks is spoiled."""
    B, T, HQ, D = q.shape
    H, dev, scale = cache.kv_heads, out.device, D ** -0.5
    K, V = contents(cache)
    for b, n in enumerate(lengths):
        K[b, :, n + counts[b]:], V[b, :, n + counts[b]:] = 0, 0
    most = cache.slots * np.abs(V).max()
    for b in range(B):
        see = O.visible(lengths[b], counts[b], T, cache.slots, "mask", masks[b].numpy(), window, sinks,
                        positions[b].numpy())
        see = torch.tensor(see).to(dev)[:, None, None]
        k, v = (torch.tensor(x[b]).to(dev) for x in (K, V))
        rows = q[b].double().to(dev).view(T, H, HQ // H, D).permute(1, 0, 2, 3).reshape(H, -1, D)

        def product(x, y):
            return torch.bmm(x, y.contiguous()).view(H, T, HQ // H, -1).permute(1, 0, 2, 3)

        x = (product(rows, k.transpose(1, 2)) * scale).masked_fill(~see, -INF)
        mass = (product(rows.abs(), k.abs().transpose(1, 2)) * scale).masked_fill(~see, 0).amax(-1)
        rl = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(rl > -INF, rl, torch.zeros_like(rl))[..., None])
        p = p.permute(1, 0, 2, 3).reshape(H, -1, cache.slots)
        ro, weight = product(p, v), product(p, v.abs())
        got, o = lse[b].double().view(T, H, -1), out[b].double().view(T, H, -1, D)
        f = rl > -INF
        assert torch.equal(got == -INF, ~f) and not o[~f].any(), b
        err = mass * 2.0 ** -16
        assert torch.all((got - rl)[f].abs() <= (err + 2.0 ** -20 * (1 + rl.abs()))[f]), b
        lo, hi = O.output_range(ro.cpu().numpy(), weight.cpu().numpy(), err.cpu().numpy(), dtype, most)
        o, f = o.cpu().numpy(), f.cpu().numpy()
        assert np.all(((o >= lo) & (o <= hi))[f]), b


CASES = [
    # B, T, HQ, H, D, pages, dtype, lengths, counts
    (1, 1, 1, 1, 64, 1, "bf16", [0], None),
    (2, 9, 4, 2, 128, 4, "bf16", [120, 0], None),
    (3, 33, 10, 2, 64, 6, "f16", [300, 31, 63], [33, 20, 0]),
    (2, 64, 8, 2, 128, 5, "bf16", [130, 250], [64, 50]),
    (1, 16, 32, 8, 128, 40, "bf16", [2400], None),
    (66, 5, 4, 1, 64, 3, "f16", [2 * b for b in range(66)], None),
    # one, four and eight row tiles a workgroup
    (32, 8, 32, 8, 128, 4, "bf16", [7 * b % 240 for b in range(32)], None),
    (32, 32, 32, 8, 64, 4, "f16", [7 * b % 220 for b in range(32)], [1 + b for b in range(32)]),
    (32, 64, 32, 8, 128, 4, "bf16", [6 * b for b in range(32)], None),
]


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (5, 4), (20, 70), (64, 64), (100, 300), (500, 3)])
@pytest.mark.parametrize("B,T,HQ,H,D,pages,dtype,lengths,counts", CASES)
def test_rows_of_a_tree_see_by_their_positions(pkg, dev, B, T, HQ, H, D, pages, dtype, lengths, counts, window, sinks):
    say("positions", B, T, HQ, H, D, dtype, window, sinks)
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, "causal", lengths, counts, seed=B + T)
    masks, positions = trees(B, T, T + window, lengths)
    mine = cache.block_table.clone()
    spare = sorted(set(range(cache.data.shape[0])) - set(mine.cpu().flatten().tolist()))
    for b, n in enumerate(lengths):                                # pages that no row sees: none, or one of NaN
        for i, p in enumerate(range(-(-sinks // 64), max(0, n - window + 1) // 64)):
            cache.block_table[b, p] = (-1, spare[0], 10 ** 9)[i % 3]
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), block=masks.to(dev), counts=ints(counts, dev),
                                 window=window, sinks=sinks, positions=positions.to(dev))
    torch.cuda.synchronize()
    cache.block_table.copy_(mine)
    check(cache, q, masks, positions, lengths, counts or [T] * B, window, sinks, out, lse, dtype)


@pytest.mark.parametrize("window,sinks", [(3, 0), (3, 2), (40, 4), (200, 0)])
def test_a_branch_of_a_tree_is_what_decoding_it_alone_gives(pkg, dev, window, sinks):
    """A tree's rows, rotated and windowed by positions, against each branch appended and attended by itself.

    Keys and values are multiples of 2^-3 below 2, which every block holds as they are, and the
    rotation is by quarter turns: both caches hold the same numbers, and so the same range holds both outputs.
    """
    say("branches", window, sinks)
    HQ, H, D, T, n = 4, 2, 64, 24, 150
    g = torch.Generator().manual_seed(window)
    turn = torch.arange(400) % 4
    cos = torch.tensor([1.0, 0.0, -1.0, 0.0])[turn][:, None].expand(400, D // 2).contiguous().to(dev)
    sin = torch.tensor([0.0, 1.0, 0.0, -1.0])[turn][:, None].expand(400, D // 2).contiguous().to(dev)
    rotary = pkg.RotaryTable(cos, sin)

    def rows(count, heads):
        x = torch.randint(-15, 16, (1, count, heads, D), generator=g).float() / 8
        return x.to(torch.bfloat16).to(dev)

    k, v, q = rows(n + T, H), rows(n + T, H), rows(T, HQ)
    bits, depth = tree(T, np.random.default_rng(5))
    positions = torch.tensor([[n + d for d in depth]], dtype=torch.int32, device=dev)
    masks = torch.tensor([bits], dtype=torch.int64, device=dev)
    cache, alone = (pkg.KV8Cache.allocate(1, 256, H, D, dev) for _ in "ab")
    for c in (cache, alone):
        pkg.kv8_append(c, k[:, :n], v[:, :n], ints([0], dev), rotary=rotary)
    at = ints([n], dev)
    turned = pkg.kv8_append(cache, k[:, n:], v[:, n:], at, rotary=rotary, positions=positions, q=q)
    out, lse = pkg.kv8_attention(turned, cache, at, block=masks, window=window, sinks=sinks, positions=positions)
    depths = set()
    for t in range(T):
        path = [i for i in range(T) if bits[t] >> i & 1]
        m = len(path)
        depths.add(m)
        pick = torch.tensor(path, device=dev)
        row = pkg.kv8_append(alone, k[:, n:][:, pick].contiguous(), v[:, n:][:, pick].contiguous(), at, rotary=rotary,
                             q=q[:, pick].contiguous())
        torch.cuda.synchronize()
        assert torch.equal(row[:, -1], turned[:, t])
        one, l1 = pkg.kv8_attention(row[:, -1:].contiguous(), alone, ints([n + m - 1], dev), window=window, sinks=sinks)
        torch.cuda.synchronize()
        K, V = contents(alone)
        K[:, :, n + m:], V[:, :, n + m:] = 0, 0
        ro, rl, weight, mass = O.attention(row[:, -1:].double().cpu().numpy(), K, V, [n + m - 1], [1], "causal",
                                           D ** -0.5, None, window, sinks)
        err = mass * 2.0 ** -16
        lo, hi = O.output_range(ro, weight, err, "bf16", V.shape[2] * np.abs(V).max())
        for o, l in ((out[:, t:t + 1], lse[:, t:t + 1]), (one, l1)):
            o, l = o.double().cpu().numpy(), l.double().cpu().numpy()
            assert np.all(np.abs(l - rl) <= err + 2.0 ** -20 * (1 + np.abs(rl))), t
            assert np.all((o >= lo) & (o <= hi)), t
    assert max(depths) > 3 and len(depths) < T                     # a tree: rows lie behind their depths


def test_positions_out_of_range_one_row_for_all_and_blocks_in_a_row(pkg, dev):
    """Positions outside the block's count as the nearest inside; one row of them is a stride of zero; consecutive
    ones are what the slots say."""
    say("odd positions")
    B, T, HQ, H, D, n = 3, 12, 4, 2, 64, 100
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, 3, "bf16", "mask", [n] * B, None, 7)
    lengths, qd, md = ints([n] * B, dev), q.to(dev), masks.to(dev)
    wild = torch.tensor([-2 ** 31, 0, n - 1, n, n + 3, n + T - 1, n + T, 2 ** 31 - 1, n + 5, 7, n + 2, n + 2],
                        dtype=torch.int32)
    for window, sinks in ((4, 0), (7, 103), (60, 2)):
        kw = dict(block=md, window=window, sinks=sinks)
        rows = wild[None].repeat(B, 1)
        got = pkg.kv8_attention(qd, cache, lengths, positions=rows.to(dev), **kw)
        one = pkg.kv8_attention(qd, cache, lengths, positions=wild[None].to(dev).expand(B, T), **kw)
        torch.cuda.synchronize()
        check(cache, q, masks, rows, [n] * B, [T] * B, window, sinks, *got, "bf16")
        assert torch.equal(got[0], one[0]) and torch.equal(got[1], one[1])
        wide = torch.zeros(B, 3 * T, dtype=torch.int32, device=dev)
        wide[:, T:2 * T] = n + torch.arange(T, device=dev)
        own = pkg.kv8_attention(qd, cache, lengths, positions=wide[:, T:2 * T], **kw)
        plain = pkg.kv8_attention(qd, cache, lengths, **kw)
        torch.cuda.synchronize()
        check(cache, q, masks, wide[:, T:2 * T].cpu(), [n] * B, [T] * B, window, sinks, *own, "bf16")
        assert torch.equal(own[1], plain[1]) and torch.equal(own[0], plain[0])


def test_positions_in_a_graph(pkg, dev):
    """Captured once, replayed on new queries, trees, positions and lengths, with eager calls between."""
    say("positions in a graph")
    B, T, HQ, H, D, pages = 4, 20, 8, 2, 128, 30
    cache = random_cache(pkg, dev, B, H, D, pages, seed=3)
    q = torch.zeros(B, T, HQ, D, dtype=torch.bfloat16, device=dev)
    masks, positions = (torch.zeros(B, T, dtype=x, device=dev) for x in (torch.int64, torch.int32))
    lengths = positions[:, 0].clone()

    def call():
        return pkg.kv8_attention(q, cache, lengths, block=masks, window=300, sinks=4, positions=positions) + \
            pkg.kv8_attention(q, cache, lengths, block=masks, window=6, positions=positions)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    g = torch.Generator().manual_seed(1)
    for i in range(6):
        n = [(400 * i + 301 * b) % (64 * pages - T) for b in range(B)]
        m, p = trees(B, T, i, n)
        q.copy_(torch.randn(q.shape, generator=g))
        lengths.copy_(torch.tensor(n)), masks.copy_(m), positions.copy_(p)
        eager = call()
        for _ in range(2):
            for x in captured:
                x.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(captured, eager):
                assert torch.equal(x, y), i


@pytest.mark.parametrize("given", ["slots", "own", "one row"])
def test_append_by_positions_writes_its_blocks_and_nothing_else(pkg, dev, given):
    """Positions inside and outside the table: the oracle's blocks, and every other page as it was before the call."""
    say("append by positions", given)
    B, T, H, G, D = 3, 5, 2, 2, 64
    k, v, q = append_inputs(B, T, H, G, D, "bf16", False, 8)
    cos, sin = tables(50, 32, dev)
    lengths = [0, 20, 47]
    own = torch.tensor([[0, 1, 1, 2, 49], [3, 50, -1, 2 ** 31 - 1, -2 ** 31], [7, 7, 7, 7, 7]], dtype=torch.int32)
    at = {"slots": None, "own": own.to(dev), "one row": own[1:2].to(dev).expand(B, T)}[given]
    p = np.array(lengths)[:, None] + np.arange(T) if at is None else at.cpu().numpy().astype(np.int64)
    cache = random_cache(pkg, dev, B, H, D, 2, seed=4)
    before, spare = unpacked(cache), cache.data.cpu().numpy().copy()
    turned = pkg.kv8_append(cache, k.to(dev), v.to(dev), ints(lengths, dev), positions=at, q=q.to(dev),
                            rotary=pkg.RotaryTable(cos, sin))
    torch.cuda.synchronize()
    kt = np.stack([O.rotate(k.float().numpy()[:, :, h], cos.cpu().numpy(), sin.cpu().numpy(), p, False)
                   for h in range(H)], 2)
    values = v.float().numpy()
    check_append(cache, before, spare, kt, values, lengths, None)
    # the check itself notices a byte that changed in a page that no row of the table names
    named = set(cache.block_table.cpu().flatten().tolist())
    stray = spare.copy()
    stray[next(i for i in range(len(spare)) if i not in named), 1, 77] ^= 1
    with pytest.raises(AssertionError):
        check_append(cache, before, stray, kt, values, lengths, None)
    # a query at a position that the table does not have: its rotated channels are NaN, the others are kept,
    # and all that it sees it scores NaN
    lost = torch.tensor((p < 0) | (p >= 50))
    assert lost.any() or given == "slots" and not lost[:2].any()
    nan = turned.cpu().isnan()
    assert torch.equal(nan[..., :32], lost[:, :, None, None].expand(B, T, H * G, 32)) and not nan[..., 32:].any()
    assert torch.equal(turned.cpu()[..., 32:], q[..., 32:])
    _, lse = pkg.kv8_attention(turned, cache, ints(lengths, dev), block="none")
    torch.cuda.synchronize()
    seen = torch.tensor(lengths)[:, None].expand(B, T) > 0
    assert torch.equal(lse.cpu().isnan(), (lost & seen)[..., None].expand(B, T, H * G))


@pytest.mark.parametrize("pages,columns", [(0, 3), (3, 0)])
def test_positions_over_caches_of_nothing(pkg, dev, pages, columns):
    """No pages, or a table of no columns: every row sees nothing, whatever its position."""
    say("positions and nothing", pages, columns)
    cache = pkg.KV8Cache(torch.zeros(pages, 2, 8320, dtype=torch.uint8, device=dev),
                         torch.zeros(2, columns, dtype=torch.int32, device=dev), 64)
    q = torch.randn(2, 9, 4, 64, device=dev).to(torch.bfloat16)
    masks, positions = trees(2, 9, 1, [100, 0])
    for window in (1, 5, 9):
        out, lse = pkg.kv8_attention(q, cache, ints([100, 0], dev), block=masks.to(dev), window=window, sinks=70,
                                     positions=positions.to(dev), weight_parts=2)
        torch.cuda.synchronize()
        assert not out.any() and torch.all(lse == -INF)


def test_positions_on_another_stream_with_a_workspace_of_the_callers(pkg, dev):
    say("positions on a side stream")
    B, T, HQ, H, D = 3, 14, 8, 2, 128
    lengths = [1500, 20, 700]
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, 26, "bf16", "causal", lengths, None, 3)
    masks, positions = (x.to(dev) for x in trees(B, T, 4, lengths))
    n, qd = ints(lengths, dev), q.to(dev)
    ws = pkg.ops.new_workspace(dev, 1 << 24)
    want = pkg.kv8_attention(qd, cache, n, block=masks, window=90, sinks=3, positions=positions)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [pkg.kv8_attention(qd, cache, n, block=masks, window=90, sinks=3, positions=positions, workspace=ws)
               for _ in range(3)]
    side.synchronize()
    check(cache, q, masks.cpu(), positions.cpu(), lengths, [T] * B, 90, 3, *want, "bf16")
    for o, l in got:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])
