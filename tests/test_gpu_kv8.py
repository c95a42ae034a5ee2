"""GPU tests of the 8-bit key/value cache against its 64-bit oracle.

Bounds.  What append writes and read gives back is exact: rotation and rounding are defined to the
bit.  Attention: the products of queries with codes are exact (at most 11 and 4 significant
bits) and summed in fp32, 128 terms of 2^-24 each, the factor and the scaling a few more: a score is
off by less than 2^-16 of its sum of magnitudes.  What outputs may be off by is derived at
oracle.kv8.output_range.
"""

import numpy as np
import pytest
import torch

from oracle import kv8 as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAN, INF = float("nan"), float("inf")


def say(*a):
    print("case", *a, flush=True)


def ints(x, dev):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


def random_cache(pkg, dev, B, H, D, pages, seed, spare=3):
    """A cache of random codes in shuffled pages; unnamed pages are NaN patterns throughout."""
    g = torch.Generator().manual_seed(seed)
    N = B * pages + spare
    data = torch.randint(0, 256, (N, H, O.page_bytes(D)), generator=g, dtype=torch.uint8)
    data = torch.where((data & 127) == 127, data ^ 1, data)
    data[..., 128 * D:] = 0
    for at in (0, 1, 8, 9):
        data[..., 128 * D + at] = torch.randint(116, 122, (N, H), generator=g, dtype=torch.uint8)
    table = torch.randperm(N, generator=g)[:B * pages].view(B, pages).int()
    unused = sorted(set(range(N)) - set(table.flatten().tolist()))
    data[unused] = 255
    return pkg.KV8Cache(data.to(dev), table.to(dev), D)


def spoil(cache, ends):
    """NaN codes in every slot from ends[b] on, and NaN exponents of the blocks that hold nothing below."""
    D, data, table = cache.head_dim, cache.data.cpu(), cache.block_table.cpu()
    c = torch.arange(D)
    for b, n in enumerate(ends):
        for j in range(n, cache.slots):
            page, u, s = int(table[b, j // 64]), j // 32 % 2, j % 32
            data[page][:, 32 * D * u + 16 * O.place(s) + 512 * (c // 16) + c % 16] = 255
            data[page][:, 64 * D + 32 * D * u + 16 * D * (s // 16) + s % 16 + 16 * c] = 127
            if s == 0:
                data[page][:, 128 * D + 8 * u:128 * D + 8 * u + 8] = 255
    cache.data.copy_(data)


def unpacked(cache):
    return O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), cache.head_dim)


def contents(cache):
    """64-bit keys and values [B, H, slots, D]; NaN where a row was not finite."""
    kc, ke, vc, ve, bad = unpacked(cache)
    return O.values(kc, ke, bad), O.values(vc, ve, bad)


def tables(positions, channels, dev, seed=3):
    angle = torch.rand(positions, channels // 2, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    angle = angle * 1000
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


def same(got, want):
    """Equal numbers, NaN where NaN is."""
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


# ---- append and read ---------------------------------------------------------------

APPEND = [
    # B, T, H, G, D, dtype, lengths, counts, heads first, rotated channels, interleaved
    (1, 1, 1, 1, 64, "bf16", [0], None, False, 64, False),
    (3, 1, 2, 4, 128, "f32", [0, 63, 64], None, False, 128, False),
    (2, 7, 3, 2, 128, "bf16", [1, 62], None, True, 64, True),
    (3, 16, 2, 4, 64, "f16", [5, 8, 120], [16, 0, 9], False, 16, False),
    (2, 130, 1, 3, 128, "f16", [61, 3], [130, 129], True, 0, False),
    (2, 65, 2, 1, 64, "f32", [180, 0], None, False, 32, True),     # the first runs past the table's slots
    (2, 33, 1, 5, 128, "bf16", [31, 96], None, False, 112, False),
    (4, 2, 2, 2, 64, "bf16", [31, 32, 95, 33], None, True, 64, True),
]


def append_inputs(B, T, H, G, D, dtype, heads_first, seed):
    g = torch.Generator().manual_seed(seed)

    def rows(heads):
        shape = (B, heads, T, D) if heads_first else (B, T, heads, D)
        x = (torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape, generator=g))).to(DT[dtype])
        return x.transpose(1, 2) if heads_first else x

    return rows(H), rows(H), rows(H * G)


def check_append(cache, before, spare, k, v, lengths, counts):
    """The cache's named blocks as the oracle makes them of `before`, and nothing else changed."""
    after = unpacked(cache)
    T = k.shape[1]
    for b, n in enumerate(lengths):
        count = T if counts is None else counts[b]
        state = [x[b] for x in before]
        O.append(state, k[b], v[b], n, count)
        end = min(n + count, cache.slots)
        behind = -(-end // 32) * 32 if end > n else end              # the last block's end
        for i, (got, want) in enumerate(zip(after, state)):
            got, want = got[b].copy(), want.copy()
            if want.shape[1] == cache.slots:
                # slots behind the rows in their last block may hold anything, but values of a block
                # that was written from its first row on are 0 there
                if i == 2 and end > n and max(n, behind - 32) % 32 == 0:
                    assert not got[:, end:behind].any()
                got[:, end:behind], want[:, end:behind] = 0, 0
            assert np.array_equal(got, want), b
    data = cache.data.cpu().numpy()
    named = set(cache.block_table.cpu().flatten().tolist())
    rest = [p for p in range(data.shape[0]) if p not in named]
    assert np.array_equal(data[rest], spare[rest])


@pytest.mark.parametrize("B,T,H,G,D,dtype,lengths,counts,heads_first,rot,interleaved", APPEND)
def test_append_writes_the_oracles_blocks_and_nothing_else(pkg, dev, B, T, H, G, D, dtype, lengths, counts,
                                                           heads_first, rot, interleaved):
    say("append", B, T, H, G, D, dtype, lengths, rot, interleaved)
    cache = random_cache(pkg, dev, B, H, D, 4 if T > 64 else 3, seed=T)
    k, v, q = append_inputs(B, T, H, G, D, dtype, heads_first, T + 1)
    if T > 3:                                                    # rows that are not held, and rows of zeros
        k[:, 2, 0, 3], v[:, 1, 0, 5], v[:, 3] = NAN, INF, 0
    before, spare = unpacked(cache), cache.data.cpu().numpy().copy()
    n = ints(lengths, dev)
    kd, vd, qd = (x.to(dev) for x in (k, v, q))
    kw = dict(counts=ints(counts, dev))
    turned = k.float().numpy()
    if rot:
        cos, sin = tables(260, rot, dev)
        qr = pkg.kv8_append(cache, kd, vd, n, rotary=pkg.RotaryTable(cos, sin, interleaved), q=qd, **kw)
        at = np.array(lengths)[:, None] + np.arange(T)
        c, s = cos.cpu().numpy(), sin.cpu().numpy()
        turned = np.stack([O.rotate(k.float().numpy()[:, :, h], c, s, at, interleaved) for h in range(H)], 2)
        want = np.stack([O.rotate(q.float().numpy()[:, :, h], c, s, at, interleaved) for h in range(H * G)], 2)
        for b, m in enumerate(counts or []):
            want[b, m:] = 0
        torch.cuda.synchronize()
        assert same(qr.cpu(), torch.tensor(want).to(DT[dtype]))
    else:
        assert pkg.kv8_append(cache, kd, vd, n, **kw) is None
        torch.cuda.synchronize()
    check_append(cache, before, spare, turned, v.float().numpy(), lengths, counts)


@pytest.mark.parametrize("B,T,H,G,D,dtype,lengths,counts,heads_first,rot,interleaved", APPEND)
def test_read_gives_the_values_of_slots(pkg, dev, B, T, H, G, D, dtype, lengths, counts, heads_first, rot,
                                        interleaved):
    say("read", B, T, H, D, dtype, lengths)
    cache = random_cache(pkg, dev, B, H, D, 3, seed=T + 50)
    bad = torch.randint(0, 256, (cache.data.shape[0], H, 2, 4), dtype=torch.uint8,
                        generator=torch.Generator().manual_seed(T))
    for u in (0, 1):
        cache.data[..., 128 * D + 8 * u + 4:128 * D + 8 * u + 8] = bad[:, :, u].to(dev)
    K, V = contents(cache)
    k, v = pkg.kv8_read(cache, ints(lengths, dev), T, counts=ints(counts, dev), dtype=DT[dtype])
    torch.cuda.synchronize()
    assert k.shape == v.shape == (B, T, H, D) and k.dtype == v.dtype == DT[dtype]
    want = np.zeros((2, B, T, H, D))
    for b in range(B):
        for t in range(T if counts is None else counts[b]):
            if lengths[b] + t < cache.slots:
                want[:, b, t] = K[b, :, lengths[b] + t], V[b, :, lengths[b] + t]
    for got, x in zip((k, v), want):
        assert same(got.cpu(), torch.tensor(x).float().to(DT[dtype]))


@pytest.mark.parametrize("D,step", [(64, 1), (128, 1), (128, 5)])
def test_rows_one_after_the_other(pkg, dev, D, step):
    """Rows of rising and falling size, one call each: kept rows are rounded again at every larger exponent."""
    say("append in steps", D, step)
    H, n = 2, 90
    cache = pkg.KV8Cache.allocate(1, 128, H, D, dev)
    g = torch.Generator().manual_seed(step)
    size = torch.exp2(torch.randint(-12, 12, (1, n, H, 1), generator=g).float())
    k, v = (torch.randn(1, n, H, D, generator=g) * size for _ in "kv")
    k[0, 40, 1] = NAN
    state = [x[0] for x in unpacked(cache)]
    for t in range(0, n, step):
        pkg.kv8_append(cache, k[:, t:t + step].to(dev), v[:, t:t + step].to(dev), ints([t], dev))
        O.append(state, k[0, t:t + step].numpy(), v[0, t:t + step].numpy(), t, min(step, n - t))
    torch.cuda.synchronize()
    for got, want in zip(unpacked(cache), state):
        assert np.array_equal(got[0], want)
    # rows that were rejected are written over from a shorter length; the block's exponent stays
    pkg.kv8_append(cache, k[:, :3].to(dev), v[:, :3].to(dev), ints([70], dev))
    O.append(state, k[0, :3].numpy(), v[0, :3].numpy(), 70, 3)
    torch.cuda.synchronize()
    for got, want in zip(unpacked(cache), state):
        at = slice(0, 73) if want.shape[1] == 128 else slice(0, 3)
        assert np.array_equal(got[0][:, at], want[:, at])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_rounds_ties_and_their_neighbours(pkg, dev, dtype):
    """Values at every middle of two levels, one unit of their type to either side, at many exponents."""
    say("append ties", dtype)
    D = 128
    mids = torch.tensor(np.concatenate([O.MIDDLES, O.LEVELS])).float()
    x = torch.stack([mids, torch.nextafter(mids, torch.full_like(mids, 1e9)), torch.nextafter(mids, -mids)])
    x = torch.cat([x.flatten(), torch.full((1024 - x.numel(),), 3.0)]).view(8, D)
    rows = []
    for e in (-14, -9, -3, 0, 2, 7) if dtype != "f16" else (-9, -3, 0, 2, 7):
        y = torch.cat([x, -x, torch.zeros(16, D)]) * 2.0 ** e      # a block each
        y[16:] = 448.0 * 2.0 ** e                                  # and its exponent
        rows.append(y)
    k = torch.cat(rows).to(DT[dtype])[None, :, None]
    if dtype != "f32":                                             # one unit of 16 bits to either side
        bits = k.view(torch.int16)
        bits[0, 1::3] += 1
        bits[0, 2::3] -= 1
        k = torch.where(k.isfinite(), k, torch.zeros_like(k))
    # the largest may now be over 448 times a power of two
    v = k.flip(1).contiguous()
    n = k.shape[1]
    cache = pkg.KV8Cache.allocate(1, n, 1, D, dev)
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    torch.cuda.synchronize()
    state = [np.zeros_like(x[0]) for x in unpacked(cache)]
    O.append(state, k[0].float().numpy(), v[0].float().numpy(), 0, n)
    for got, want in zip(unpacked(cache), state):
        assert np.array_equal(got[0][:, :n], want[:, :n])


def test_exponents_at_their_borders(pkg, dev):
    """A block's largest magnitude at 448 times a power of two and one float to either side, very small and large."""
    say("exponents")
    D, tops = 64, []
    for e in (-70, -64, -63, -20, 0, 5, 30, 62, 63, 64):
        x = np.float32(448.0 * 2.0 ** e)
        tops += [x, np.nextafter(x, np.float32(0)), np.nextafter(x, np.float32(np.inf))]
    tops += [0.0, 1e-45, 1e-38, 3.0e38]
    n = 32 * len(tops)
    k = torch.zeros(1, n, 1, D)
    for i, x in enumerate(tops):
        k[0, 32 * i + i % 32, 0, i % D] = float(x)
        k[0, 32 * i + (i + 1) % 32, 0, 3] = float(x) / 3
    cache = pkg.KV8Cache.allocate(1, n, 1, D, dev)
    pkg.kv8_append(cache, k.to(dev), (-k).to(dev), ints([0], dev))
    torch.cuda.synchronize()
    state = [np.zeros_like(x[0]) for x in unpacked(cache)]
    O.append(state, k[0].numpy(), -k[0].numpy(), 0, n)
    for got, want in zip(unpacked(cache), state):
        assert np.array_equal(got[0][:, :want.shape[1]], want)
    assert state[4].any() and not state[4].all()


def test_positions_are_given_or_the_slots(pkg, dev):
    """Positions of their own (a tree's depths), one row for all, and positions that the table does not have."""
    say("positions")
    B, T, H, G, D = 3, 5, 2, 2, 64
    k, v, q = append_inputs(B, T, H, G, D, "bf16", False, 8)
    cos, sin = tables(50, 32, dev)
    wide = torch.zeros(50, 2, 16, device=dev)
    wide[:, 0], wide[:, 1] = cos, sin
    rotary = pkg.RotaryTable(wide[:, 0], wide[:, 1])               # rows of both in one tensor
    lengths = [0, 20, 47]
    own = torch.tensor([[0, 1, 1, 2, 49], [3, 50, -1, 2 ** 31 - 1, -2 ** 31], [7, 7, 7, 7, 7]], dtype=torch.int32)
    for at in (None, own, own[:1].expand(B, T)):
        cache = random_cache(pkg, dev, B, H, D, 2, seed=4)
        before = unpacked(cache)
        qin = q.to(dev)
        out = pkg.kv8_append(cache, k.to(dev), v.to(dev), ints(lengths, dev), rotary=rotary, q=qin, q_out=qin,
                             positions=None if at is None else (at.to(dev) if at.stride(0) else
                                                                at[:1].to(dev).expand(B, T)))
        torch.cuda.synchronize()
        assert out is qin
        p = np.array(lengths)[:, None] + np.arange(T) if at is None else at.numpy().astype(np.int64)
        c, s = cos.cpu().numpy(), sin.cpu().numpy()
        kt = np.stack([O.rotate(k.float().numpy()[:, :, h], c, s, p, False) for h in range(H)], 2)
        qt = np.stack([O.rotate(q.float().numpy()[:, :, h], c, s, p, False) for h in range(H * G)], 2)
        assert same(out.cpu(), torch.tensor(qt).to(torch.bfloat16))
        check_append(cache, before, cache.data.cpu().numpy(), kt, v.float().numpy(), lengths, None)
        lost = unpacked(cache)[4]
        assert lost.any() == bool(((p < 0) | (p >= 50)).any())


# ---- attention -----------------------------------------------------------------------

ATTENTION = [
    # B, T, HQ, H, D, pages, dtype, block, lengths, counts
    (1, 1, 1, 1, 64, 1, "bf16", "causal", [0], None),
    (2, 1, 8, 2, 128, 3, "bf16", "causal", [130, 1], None),
    (3, 4, 4, 4, 64, 2, "f16", "full", [0, 64, 100], [4, 1, 0]),
    (2, 5, 12, 4, 128, 12, "f16", "causal", [700, 3], None),
    (1, 16, 32, 8, 128, 40, "bf16", "causal", [2400], None),
    (2, 33, 10, 2, 64, 10, "f16", "mask", [500, 31], [33, 20]),
    (4, 64, 4, 1, 128, 3, "bf16", "mask", [0, 63, 64, 90], None),
    (2, 7, 6, 2, 64, 4, "bf16", "none", [200, 0], None),
    (2, 70, 8, 2, 128, 5, "bf16", "causal", [250, 0], [70, 69]),
    (1, 300, 8, 2, 64, 7, "f16", "causal", [100], None),
    (1, 3, 64, 1, 128, 3, "bf16", "full", [150], None),
    (3, 2, 3, 1, 64, 66, "bf16", "causal", [4200, 2000, 64], None),
]
# window, sinks
WINDOWS = [(1, 0), (1, 1), (40, 4), (64, 64), (97, 130), (1000, 3), (5000, 0)]


def attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed, sharp=1.0):
    cache = random_cache(pkg, dev, B, H, D, pages, seed)
    ends = [n if block == "none" else min(n + (T if counts is None else counts[b]), 64 * pages)
            for b, n in enumerate(lengths)]
    spoil(cache, ends)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(B, T, HQ, D, generator=g) * sharp).to(DT[dtype])
    masks = torch.randint(-2 ** 63, 2 ** 63 - 1, (B, T), generator=g) if block == "mask" else None
    return cache, q, masks


def check_attention(cache, q, dtype, block, lengths, counts, masks, scale, out, lse, window=None, sinks=0, steep=False):
    K, V = contents(cache)
    B, T = q.shape[:2]
    count = [min(T if counts is None else counts[b], T) for b in range(B)]
    for b, n in enumerate(lengths):                                # what was spoiled is not there
        end = n if block == "none" else n + count[b]
        K[b, :, end:], V[b, :, end:] = 0, 0
    ro, rl, weight, mass = O.attention(q.double().numpy(), K, V, lengths, count, block, scale,
                                       None if masks is None else masks.numpy(), window, sinks)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    lost = np.isnan(rl)
    assert np.array_equal(lost, np.isnan(lse)) and np.all(np.isnan(out[lost]))
    empty = np.isneginf(rl)
    assert np.array_equal(empty, np.isneginf(lse)) and np.all(out[empty] == 0)
    f = ~empty & ~lost
    err = mass * 2.0 ** -16
    with np.errstate(invalid="ignore"):
        assert np.all(np.abs(lse - rl)[f] <= (err + 2.0 ** -20 * (1 + np.abs(rl)))[f])
        # steep: no weight that matters is so small that it has fewer bits
        most = 0.0 if steep else V.shape[2] * np.nanmax(np.abs(V), initial=0.0)
        lo, hi = O.output_range(ro, weight, err, dtype, most)
    ok = (out >= lo) & (out <= hi)
    assert ok[f].all(), (np.argwhere(~ok & f[..., None])[:4], out[~ok & f[..., None]][:4], ro[~ok & f[..., None]][:4])


@pytest.mark.parametrize("B,T,HQ,H,D,pages,dtype,block,lengths,counts", ATTENTION)
def test_attention_matches_oracle(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts):
    say("attention", B, T, HQ, H, D, pages, dtype, block, lengths, counts)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed=B * T)
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev),
                                 block=block if masks is None else masks.to(dev), counts=ints(counts, dev))
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    check_attention(cache, q, dtype, block, lengths, counts, masks, D ** -0.5, out, lse)


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("B,T,HQ,H,D,pages,dtype,block,lengths,counts", ATTENTION)
def test_windows_match_oracle(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, window, sinks):
    """Entries of pages that no row sees name none, or a page of NaN: nothing of them arrives."""
    say("window", window, sinks, B, T, HQ, H, D, pages, dtype, block, lengths, counts)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed=B + T)
    mine = cache.block_table.clone()
    spare = sorted(set(range(cache.data.shape[0])) - set(mine.cpu().flatten().tolist()))
    for b, n in enumerate(lengths):
        gone = range(-(-sinks // 64), max(0, n - window + 1) // 64)
        for i, p in enumerate(gone):
            cache.block_table[b, p] = (-1, spare[0], 10 ** 9)[i % 3]
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), window=window, sinks=sinks,
                                 block=block if masks is None else masks.to(dev), counts=ints(counts, dev))
    torch.cuda.synchronize()
    cache.block_table.copy_(mine)
    check_attention(cache, q, dtype, block, lengths, counts, masks, D ** -0.5, out, lse, window, sinks)


@pytest.mark.parametrize("sharp,scale", [(40.0, None), (1e-3, 1.0), (1.0, -2.0), (1.0, 0.0), (1.0, 1e-30)])
def test_attention_over_sharp_flat_and_negative_scores(pkg, dev, sharp, scale):
    """Scores of several hundred (one slot takes all), of nearly nothing, and scales that are not positive."""
    say("attention scores", sharp, scale)
    cache, q, _ = attention_inputs(pkg, dev, 2, 6, 8, 2, 128, 6, "bf16", "causal", [300, 40], None, 5, sharp)
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints([300, 40], dev), scale=scale)
    torch.cuda.synchronize()
    check_attention(cache, q, "bf16", "causal", [300, 40], None, None, 128 ** -0.5 if scale is None else scale,
                    out, lse)


def test_attention_rising_scores(pkg, dev):
    """Every slot's score exceeds those before it by more: the running maximum moves on at every step."""
    say("attention rising")
    D, n = 64, 500
    cache = pkg.KV8Cache.allocate(1, 512, 1, D, dev)
    k = torch.zeros(1, n, 1, D)
    k[0, :, 0, 0] = torch.linspace(-60, 60, n)
    v = torch.randn(1, n, 1, D, generator=torch.Generator().manual_seed(1))
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16)
    q[0, 0, 0, 0], q[0, 1, 0, 0] = 3.0, -3.0
    for window in (None, 100):
        out, lse = pkg.kv8_attention(q.to(dev), cache, ints([n], dev), block="none", scale=1.0, window=window)
        torch.cuda.synchronize()
        check_attention(cache, q, "bf16", "none", [n], None, None, 1.0, out, lse, window)


@pytest.mark.parametrize("T,n,dtype,step", [(1, 700, "bf16", 0.0), (3, 700, "bf16", 0.01), (40, 300, "bf16", 0.02),
                                            (2, 5000, "f16", 0.001)])
def test_values_up_to_what_the_cache_holds(pkg, dev, T, n, dtype, step):
    """Values of 448 * 2^64 under even weights and rising ones: no sum overflows."""
    say("large values", T, n, dtype, step)
    HQ, H, D = 4, 2, 64
    g = torch.Generator().manual_seed(n)
    cache = pkg.KV8Cache.allocate(1, n + T, H, D, dev)
    k = torch.zeros(1, n + T, H, D)
    k[0, :, :, 0] = (torch.arange(n + T) * 1.0)[:, None]
    v = torch.where(torch.rand(D, generator=g) < 0.5, -1.0, 1.0).expand(1, n + T, H, D) * O.MOST
    v = v * (0.8 + 0.2 * torch.rand(1, n + T, H, D, generator=g))
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = torch.zeros(1, T, HQ, D, dtype=DT[dtype])
    q[..., 0] = 1.0
    scale = step if step else 1e-6
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints([n], dev), scale=scale)
    torch.cuda.synchronize()
    if dtype == "f16":                                             # past the type's range, as the values are
        K, V = contents(cache)
        ref = O.attention(q.double().numpy(), K, V, [n], [T], "causal", scale)[0]
        assert np.array_equal(out.cpu().numpy(), np.sign(ref) * np.inf)
    else:
        check_attention(cache, q, dtype, "causal", [n], None, None, scale, out, lse)


@pytest.mark.parametrize("T,dtype", [(1, "bf16"), (3, "f16"), (20, "bf16"), (40, "f16")])
@pytest.mark.parametrize("up", [True, False])
def test_blocks_of_very_different_scales(pkg, dev, T, dtype, up):
    """Values from 2^-60 to 2^60, block by block, where the large ones weigh nothing: the small ones count in full."""
    say("scales", T, dtype, up)
    HQ, H, D, n = 4, 2, 64, 500
    g = torch.Generator().manual_seed(T)
    cache = pkg.KV8Cache.allocate(1, n + T, H, D, dev)
    order = torch.arange(n + T) // 32 * 7 - 55                     # binary orders of a block's values
    size = order.float() if up else -order.float() - 1
    v = torch.randn(1, n + T, H, D, generator=g) * torch.exp2(size)[None, :, None, None]
    k = torch.zeros(1, n + T, H, D)
    k[0, :, :, 0] = -size[:, None] * 1.5                           # the larger, the less it is looked at
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = torch.zeros(1, T, HQ, D, dtype=DT[dtype])
    q[..., 0] = torch.linspace(0.3, 3.0, HQ)
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints([n], dev), block="full", scale=1.0)
    torch.cuda.synchronize()
    check_attention(cache, q, dtype, "full", [n], None, None, 1.0, out, lse, steep=True)


@pytest.mark.parametrize("T,block,window", [(1, "causal", None), (9, "causal", None), (9, "mask", None),
                                            (40, "causal", 30), (12, "full", 200), (12, "full", 60)])
def test_rows_that_are_not_held(pkg, dev, T, block, window):
    """A row of NaN or infinity in the cache makes NaN of the rows that see it, and of no other."""
    say("bad rows", T, block, window)
    B, HQ, H, D, lengths = 2, 4, 2, 128, [90, 200]
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, 6, "bf16", block, lengths, None, 3)
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(B, T, H, D, generator=g) for _ in "kv")
    k[0, T // 2, 1, 5], v[1, T - 1, 0, 7] = INF, NAN
    pkg.kv8_append(cache, k.to(dev), v.to(dev), ints(lengths, dev))
    sinks = 2 if window else 0
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), window=window, sinks=sinks,
                                 block=block if masks is None else masks.to(dev))
    torch.cuda.synchronize()
    check_attention(cache, q, "bf16", block, lengths, None, masks, D ** -0.5, out, lse, window, sinks)
    assert T == 1 or block == "full" or not lse.isnan().all()
    # an old row in a page that is read whole, outside the window of all rows
    if window and window < lengths[0]:
        k[0, T // 2, 1, 5] = 1.0
        v[1, T - 1, 0, 7] = 1.0
        pkg.kv8_append(cache, k.to(dev), v.to(dev), ints(lengths, dev))
        pkg.kv8_append(cache, torch.full((B, 1, H, D), NAN, device=dev), torch.zeros(B, 1, H, D, device=dev),
                       ints([lengths[0] - window, 0], dev), counts=ints([1, 0], dev))
        out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), window=window, sinks=sinks, block=block)
        torch.cuda.synchronize()
        assert unpacked(cache)[4][0, :, lengths[0] - window].all()
        assert not lse.isnan().any() and not out.isnan().any()


@pytest.mark.parametrize("dtype,T,block", [("bf16", 3, "causal"), ("f16", 9, "full"), ("bf16", 40, "causal")])
def test_rows_of_nan_and_infinite_queries(pkg, dev, dtype, T, block):
    """Their out and lse are NaN; other rows are as ever."""
    say("nan queries", dtype, T, block)
    B, HQ, H, D, lengths, counts = 3, 4, 2, 64, [130, 700, 0], [T, T, T - 1]
    cache, q, _ = attention_inputs(pkg, dev, B, T, HQ, H, D, 12, dtype, block, lengths, counts, 17)
    bad = torch.zeros(B, T, HQ, dtype=torch.bool)
    for (b, t, hq), x in {(0, 0, 1): "nan", (0, T - 2, 0): "inf", (1, 1, 3): "-inf", (1, T - 1, 3): "nan",
                          (2, 1, 0): "nan"}.items():
        q[b, t, hq, 7 * hq + 2] = float(x)
        bad[b, t, hq] = True
    q[2, T - 1] = NAN                                              # no valid row
    n, c = ints(lengths, dev), ints(counts, dev)
    out, lse = pkg.kv8_attention(q.to(dev), cache, n, block=block, counts=c)
    torch.cuda.synchronize()
    assert torch.equal(lse.cpu().isnan(), bad)
    assert torch.equal(out.cpu().isnan(), bad[..., None].expand_as(out))
    clean = torch.where(bad[..., None] | q.isnan(), torch.zeros_like(q), q)
    o, l = out.cpu(), lse.cpu()
    co, cl = (x.cpu() for x in pkg.kv8_attention(clean.to(dev), cache, n, block=block, counts=c))
    o[bad], l[bad] = co[bad], cl[bad]
    check_attention(cache, clean, dtype, block, lengths, counts, None, D ** -0.5, o, l)


def attention_64(cache, q, n, c, block, masks, window, sinks):
    """The same products in 64 bits on the GPU, for sizes that the oracle is slow for: (out, lse, weight, mass)."""
    B, T, HQ, D = q.shape
    H, dev = cache.kv_heads, cache.device
    K, V = (torch.tensor(x).to(dev).nan_to_num() for x in contents(cache))
    see = np.stack([O.visible(n[b], c[b], T, cache.slots, block, None if masks is None else masks[b].numpy(), window,
                              sinks) for b in range(B)])
    see = torch.tensor(see).to(dev)
    q64 = q.double().to(dev).view(B, T, H, -1, D)
    for b in range(B):
        x = torch.einsum("thgd,hjd->thgj", q64[b], K[b]) * D ** -0.5
        mass = torch.einsum("thgd,hjd->thgj", q64[b].abs(), K[b].abs()) * D ** -0.5
        hidden = ~see[b][:, None, None]
        mass = mass.masked_fill(hidden, 0).amax(-1)
        x = x.masked_fill(hidden, -INF)
        rl = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(rl > -INF, rl, torch.zeros_like(rl))[..., None])
        yield (torch.einsum("thgj,hjd->thgd", p, V[b]), rl, torch.einsum("thgj,hjd->thgd", p, V[b].abs()), mass)


@pytest.mark.parametrize("B,H,T,G,D,dtype,block,ragged,pages,window", [
    (32, 8, 32, 4, 64, "bf16", "causal", True, 3, None),           # 4 row tiles
    (20, 4, 75, 3, 64, "f16", "full", False, 3, 60),               # 8, the last one of one row
    (16, 8, 64, 8, 128, "bf16", "mask", True, 3, None),            # 16
    (2, 8, 515, 4, 128, "bf16", "causal", True, 12, None),         # 65
    (1, 4, 700, 5, 128, "f16", "causal", False, 12, 150),
    (3, 2, 300, 7, 64, "bf16", "causal", False, 7, 65),
    (70, 4, 40, 4, 128, "bf16", "causal", True, 2, 33),            # more sequences than a wave's lanes
])
def test_attention_of_many_row_tiles(pkg, dev, B, H, T, G, D, dtype, block, ragged, pages, window):
    """Sizes at which a workgroup takes several row tiles: every row against 64-bit products."""
    say("attention many tiles", B, H, T, G, D, dtype, block, window)
    counts = [1 + (7 * b) % T if b else T for b in range(B)] if ragged else None
    lengths = [(13 * b + 5) % max(1, 64 * pages - T) for b in range(B)]
    cache, q, masks = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, dtype, block, lengths, counts, B)
    sinks = 3 if window else 0
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), counts=ints(counts, dev), window=window,
                                 sinks=sinks, block=block if masks is None else masks.to(dev))
    torch.cuda.synchronize()
    c = [T] * B if counts is None else counts
    most = cache.slots * np.nanmax(np.abs(contents(cache)[1]))
    for b, (ro, rl, weight, mass) in enumerate(attention_64(cache, q, lengths, c, block, masks, window, sinks)):
        err = mass * 2.0 ** -16
        got = lse[b].double().view(T, H, G)
        f = rl > -INF
        assert torch.equal(f, got > -INF)
        assert torch.all((got - rl)[f].abs() <= (err + 2.0 ** -20 * (1 + rl.abs()))[f]), b
        lo, hi = O.output_range(ro.cpu().numpy(), weight.cpu().numpy(), err.cpu().numpy(), dtype, most)
        o = out[b].double().view(T, H, G, D).cpu().numpy()
        assert np.all((o >= lo) & (o <= hi)), b


CUTS = [
    # B, T, HQ, H, pages, lengths: long ones among short ones, more tile groups than workgroups, many parts
    (3, 1, 4, 1, 130, [8000, 10, 0], None),
    (2, 2, 64, 32, 40, [2500, 1], None),
    (5, 3, 16, 16, 33, [2000, 2, 700, 64, 63], 500),
    (66, 1, 8, 4, 20, [1200] + [17 * b % 300 for b in range(65)], None),
    (1, 1, 1, 1, 300, [19000], None),
    (1, 8, 8, 1, 200, [12700], 9000),
]


@pytest.mark.parametrize("B,T,HQ,H,pages,lengths,window", CUTS)
def test_attention_of_any_cut(pkg, dev, B, T, HQ, H, pages, lengths, window):
    say("cuts", B, T, HQ, H, pages, window)
    cache = random_cache(pkg, dev, B, H, 64, pages, seed=pages)
    q = torch.randn(B, T, HQ, 64, generator=torch.Generator().manual_seed(B)).to(torch.bfloat16)
    out, lse = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), window=window, sinks=5 if window else 0)
    again = pkg.kv8_attention(q.to(dev), cache, ints(lengths, dev), window=window, sinks=5 if window else 0)
    torch.cuda.synchronize()
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    most = cache.slots * np.nanmax(np.abs(contents(cache)[1]))
    for b, (ro, rl, weight, mass) in enumerate(attention_64(cache, q, lengths, [T] * B, "causal", None, window,
                                                            5 if window else 0)):
        err = mass * 2.0 ** -16
        got = lse[b].double().view(rl.shape)
        assert torch.all((got - rl).abs() <= err + 2.0 ** -20 * (1 + rl.abs())), b
        lo, hi = O.output_range(ro.cpu().numpy(), weight.cpu().numpy(), err.cpu().numpy(), "bf16", most)
        o = out[b].double().view(ro.shape).cpu().numpy()
        assert np.all((o >= lo) & (o <= hi)), b
