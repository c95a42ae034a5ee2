"""GPU tests of the 4-bit key/value cache against its 64-bit oracle.

Bounds.  The products of queries with keys are exact and summed in fp32, so a score
is off by at most 2^-16 of its sum of magnitudes (128 terms, 2^-24 each, and the
scaling); fp16 queries meet keys held in fp16 at a sixteenth of their size, which
adds 2^-20 of the sum of |q|.  A weight p is rounded to bf16 before it meets the
values (2^-9), the output to its type (2^-9 at most): together 2^-8 of
sum p |v| / sum p, and twice the score's error.
"""

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def say(*a):
    print("case", *a, flush=True)


def random_cache(pkg, dev, B, H, D, pages, seed, spare=3):
    """A cache of random codes in shuffled pages; scales of unnamed pages are NaN patterns."""
    g = torch.Generator().manual_seed(seed)
    N = B * pages + spare
    data = torch.randint(0, 256, (N, H, O.page_bytes(D)), generator=g, dtype=torch.uint8)
    data[..., 32 * D:34 * D] = torch.randint(121, 127, (N, H, 2 * D), generator=g, dtype=torch.uint8)
    scale = (torch.rand(N, H, 64, generator=g) + 0.1).to(torch.bfloat16)
    data[..., 66 * D:] = scale.view(torch.uint8)
    table = torch.randperm(N, generator=g)[:B * pages].view(B, pages).int()
    unused = [p for p in range(N) if p not in set(table.flatten().tolist())]
    data[unused] = 255
    return pkg.KV4Cache(data.to(dev), table.to(dev), D)


def spoil(cache, lengths):
    """Fill every slot from lengths[b] on with the bits of codes -6 and scales NaN."""
    D, data = cache.head_dim, cache.data
    table = cache.block_table.cpu()
    for b, n in enumerate(lengths):
        for j in range(n, cache.slots):
            page, i = int(table[b, j // 64]), j % 64
            data[page, :, i * D // 2:(i + 1) * D // 2] = 255
            for m in range(D // 32):
                data[page, :, 32 * D + 64 * m + 16 * (i >> 3 & 3) + 4 * (i & 3) + 2 * (i >> 5) + (i >> 2 & 1)] = 255
            data[page, :, 66 * D + 2 * i:66 * D + 2 * i + 2] = 255


def contents(cache):
    """64-bit keys and values [B, H, slots, D] of the cache (non-finite scales count as 0)."""
    kc, ke, vc, vs = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), cache.head_dim)
    vs = np.where(np.isfinite(vs), vs, 0.0)
    return O.key_values(kc, np.where(ke == 255, 0, ke)), O.value_values(vc, vs)


def ints(x, dev):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


# ---- append and read ---------------------------------------------------------------

APPEND = [
    # B, T, H, D, dtype, lengths, counts, heads first
    (1, 1, 1, 64, "bf16", [0], None, False),
    (3, 1, 2, 128, "f32", [0, 63, 64], None, False),
    (2, 7, 3, 128, "bf16", [1, 62], None, True),
    (3, 16, 2, 64, "f16", [5, 8, 120], [16, 0, 9], False),
    (2, 130, 1, 128, "f16", [61, 3], [130, 129], True),
    (2, 65, 2, 64, "f32", [180, 0], None, False),          # the first runs past the table's slots
]


@pytest.mark.parametrize("B,T,H,D,dtype,lengths,counts,heads_first", APPEND)
def test_append_writes_the_oracles_codes_and_nothing_else(pkg, dev, B, T, H, D, dtype, lengths, counts, heads_first):
    say("append", B, T, H, D, dtype, lengths)
    cache = random_cache(pkg, dev, B, H, D, 4 if T > 64 else 3, seed=T)
    g = torch.Generator().manual_seed(T + 1)
    shape = (B, H, T, D) if heads_first else (B, T, H, D)
    k, v = ((torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape, generator=g))).to(DT[dtype])
            for _ in "kv")
    # rows with ties of the levels, zeros, and (where the type has them) non-finite numbers
    kt, vt = (x.transpose(1, 2) if heads_first else x for x in (k, v))
    kt[:, 0, :, :32] = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.0] * 4)
    vt[:, 0] = 0
    if T > 3:
        kt[:, 2, 0, 3], vt[:, 2, 0, 5], vt[:, 2, 0, 6] = float("nan"), float("inf"), float("nan")
    kd, vd = k.to(dev), v.to(dev)
    if heads_first:
        k, v, kd, vd = (x.transpose(1, 2) for x in (k, v, kd, vd))
    before = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), D)
    spare = cache.data.cpu().numpy().copy()
    pkg.kv4_append(cache, kd, vd, ints(lengths, dev), counts=ints(counts, dev))
    torch.cuda.synchronize()
    after = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), D)
    kc, ke = O.encode_keys(k.float().numpy())
    vc, vs = O.encode_values(v.float().numpy())
    want = [x.copy() for x in before]
    for b in range(B):
        for t in range(T if counts is None else counts[b]):
            j = lengths[b] + t
            if j < cache.slots:
                for x, y in zip(want, (kc, ke, vc, vs)):
                    x[b, :, j] = y[b, t]
    for got, x in zip(after, want):
        assert np.array_equal(got, x)
    named = set(cache.block_table.cpu().flatten().tolist())
    rest = [p for p in range(cache.data.shape[0]) if p not in named]
    assert np.array_equal(cache.data.cpu().numpy()[rest], spare[rest])


@pytest.mark.parametrize("B,T,H,D,dtype,lengths,counts,heads_first", APPEND)
def test_read_gives_the_values_of_slots(pkg, dev, B, T, H, D, dtype, lengths, counts, heads_first):
    say("read", B, T, H, D, dtype, lengths)
    cache = random_cache(pkg, dev, B, H, D, 3, seed=T + 50)
    K, V = contents(cache)
    k, v = pkg.kv4_read(cache, ints(lengths, dev), T, counts=ints(counts, dev), dtype=DT[dtype])
    torch.cuda.synchronize()
    assert k.shape == v.shape == (B, T, H, D) and k.dtype == v.dtype == DT[dtype]
    want = np.zeros((2, B, T, H, D))
    for b in range(B):
        for t in range(T if counts is None else counts[b]):
            if lengths[b] + t < cache.slots:
                want[:, b, t] = K[b, :, lengths[b] + t], V[b, :, lengths[b] + t]
    for got, x in zip((k, v), want):
        assert torch.equal(got.cpu(), torch.tensor(x).float().to(DT[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_rounds_ties_and_their_neighbours(pkg, dev, dtype):
    """Values at every threshold times their row's scale, and one unit of their type to either side."""
    say("append ties", dtype)
    D, T = 128, 600
    g = torch.Generator().manual_seed(5)
    amax = torch.exp(torch.randn(T, generator=g) * 3).clamp(1e-3, 6e4).to(DT[dtype])
    step = torch.tensor(O.encode_values(amax.float().numpy()[:, None])[1])
    mids = torch.tensor(np.concatenate([O.MIDPOINTS, -O.MIDPOINTS]))
    x = (step[:, None] * mids).to(DT[dtype])                 # a tie, where the type holds it
    bits = x.view(torch.int32 if dtype == "f32" else torch.int16)
    near = [x] + [(bits + d).view(DT[dtype]) for d in (-1, 1, -3, 3, 40, -40)]
    v = torch.cat(near + [torch.randn(T, D - 7 * 14 - 1, generator=g).to(DT[dtype]) * step[:, None].to(DT[dtype])], 1)
    v = torch.where(v.abs() > amax[:, None], torch.zeros_like(v), v)
    v = torch.cat([amax[:, None], v], 1)[None, :, None]
    cache = pkg.KV4Cache.allocate(1, T, 1, D, dev)
    pkg.kv4_append(cache, v.to(dev), v.to(dev), ints([0], dev))
    torch.cuda.synchronize()
    kc, ke, vc, vs = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), D)
    f = v[0, :, 0].float().numpy()
    for got, want in zip((kc, ke, vc, vs), (*O.encode_keys(f), *O.encode_values(f))):
        assert np.array_equal(got[0, 0, :T], want)


# ---- attention ---------------------------------------------------------------------

ATTENTION = [
    # B, T, HQ, H, D, pages, dtype, block, lengths, counts
    (1, 1, 1, 1, 64, 1, "bf16", "causal", [0], None),                 # the row sees itself alone
    (1, 1, 4, 1, 128, 2, "bf16", "causal", [63], None),
    (2, 1, 8, 2, 128, 5, "f16", "causal", [255, 17], None),
    (3, 3, 3, 3, 64, 2, "bf16", "none", [0, 1, 128], None),           # no context: an empty row
    (2, 5, 15, 3, 128, 4, "bf16", "full", [60, 192], [5, 2]),
    (3, 16, 8, 2, 128, 4, "bf16", "causal", [1, 64, 200], [16, 0, 7]),
    (2, 17, 4, 4, 64, 3, "f16", "mask", [100, 0], None),
    (1, 33, 5, 1, 64, 3, "f16", "mask", [130], None),
    (1, 9, 8, 1, 128, 2, "bf16", "causal", [60], None),               # 72 rows
    (2, 64, 2, 1, 64, 4, "bf16", "mask", [70, 3], [64, 50]),
    (1, 100, 3, 1, 128, 4, "bf16", "causal", [37], None),             # a prompt's chunk
    (2, 70, 2, 2, 64, 3, "f16", "full", [0, 90], [70, 69]),
    (1, 2, 2, 1, 128, 40, "bf16", "causal", [2500], None),            # a long axis for few rows
    (2, 4, 1, 1, 64, 3, "bf16", "causal", [190, 191], None),          # runs past the table's slots
]


def attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed, sharp=1.0):
    cache = random_cache(pkg, dev, B, H, D, pages, seed)
    count = [T] * B if counts is None else counts
    spoil(cache, [min(n + (0 if block == "none" else c), cache.slots) for n, c in zip(lengths, count)])
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(B, T, HQ, D, generator=g) * sharp).to(DT[dtype])
    masks = None
    if block == "mask":
        masks = torch.randint(-2**63, 2**63 - 1, (B, T), generator=g, dtype=torch.int64)
        masks[0, 0] = 0
    return cache, q, masks


def score_error(q, mass, dtype, scale):
    err = mass * 2.0 ** -16
    if dtype == "f16":
        err = err + np.abs(q).sum(-1) * scale * 2.0 ** -20
    return err


def check_attention(cache, q, dtype, block, lengths, counts, masks, scale, out, lse):
    K, V = contents(cache)
    B, T = q.shape[:2]
    q64 = q.double().numpy()
    # what lies past the table's slots does not exist
    count = [min(T if counts is None else counts[b], T) for b in range(B)]
    ro, rl, weight, mass = O.attention(q64, K, V, lengths, count, "mask" if masks is not None else block, scale,
                                       None if masks is None else masks.numpy())
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    err = score_error(q64, mass, dtype, scale)
    assert np.all(np.isfinite(out))
    empty = ~np.isfinite(rl)
    assert np.array_equal(empty, lse == -np.inf) and np.all(out[empty] == 0)
    tol = weight * (2.0 ** -8 * 1.01 + 2.0 * err[..., None]) + 1e-30
    worst = (np.abs(out - ro) - tol).max()
    assert worst <= 0, worst
    f = ~empty
    assert np.all(np.abs(lse[f] - rl[f]) <= err[f] + 2.0 ** -20 * (1 + np.abs(rl[f])))


@pytest.mark.parametrize("B,T,HQ,H,D,pages,dtype,block,lengths,counts", ATTENTION)
def test_attention_matches_oracle(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts):
    say("attention", B, T, HQ, H, D, pages, dtype, block, lengths, counts)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed=B * T)
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints(lengths, dev),
                                 block=block if masks is None else masks.to(dev), counts=ints(counts, dev))
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    check_attention(cache, q, dtype, block, lengths, counts, masks, D ** -0.5, out, lse)


@pytest.mark.parametrize("sharp,scale", [(40.0, None), (1e-3, 1.0), (1.0, -2.0), (1.0, 0.0)])
def test_attention_over_sharp_flat_and_negative_scores(pkg, dev, sharp, scale):
    """Scores of several hundred (one slot takes all), of nearly nothing, and scales that are not positive."""
    say("attention scores", sharp, scale)
    cache, q, _ = attention_inputs(pkg, dev, 2, 6, 8, 2, 128, 6, "bf16", "causal", [300, 40], None, 5, sharp)
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints([300, 40], dev), scale=scale)
    torch.cuda.synchronize()
    check_attention(cache, q, "bf16", "causal", [300, 40], None, None, 128 ** -0.5 if scale is None else scale,
                    out, lse)


def test_attention_rising_scores(pkg, dev):
    """Every slot's score exceeds those before it by more: the running maximum moves on at every step."""
    say("attention rising")
    D, n = 64, 500
    cache = pkg.KV4Cache.allocate(1, 512, 1, D, dev)
    k = torch.zeros(1, n, 1, D)
    k[0, :, 0, 0] = torch.linspace(-60, 60, n)
    v = torch.randn(1, n, 1, D, generator=torch.Generator().manual_seed(1))
    pkg.kv4_append(cache, k.to(dev), v.to(dev), ints([0], dev))
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16)
    q[0, 0, 0, 0], q[0, 1, 0, 0] = 3.0, -3.0
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints([n], dev), block="none", scale=1.0)
    torch.cuda.synchronize()
    check_attention(cache, q, "bf16", "none", [n], None, None, 1.0, out, lse)


@pytest.mark.parametrize("B,H,T,G,D,dtype,block,ragged", [
    (32, 8, 32, 4, 64, "bf16", "causal", True),             # 4 row tiles
    (20, 4, 75, 3, 64, "f16", "full", False),               # 8, the last one of one row
    (16, 8, 64, 8, 128, "bf16", "mask", True),              # 16
])
def test_attention_of_many_row_tiles(pkg, dev, B, H, T, G, D, dtype, block, ragged):
    """Sizes at which a workgroup takes several row tiles: every row against 64-bit products."""
    say("attention many tiles", B, H, T, G, D, dtype, block)
    pages = 3
    counts = [1 + (7 * b) % T for b in range(B)] if ragged else None
    lengths = [(13 * b + 5) % (192 - T) for b in range(B)]
    cache, q, masks = attention_inputs(pkg, dev, B, T, H * G, H, D, pages, dtype, block, lengths, counts, B)
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints(lengths, dev), counts=ints(counts, dev),
                                 block=block if masks is None else masks.to(dev))
    torch.cuda.synchronize()
    K, V = (torch.tensor(x).to(dev) for x in contents(cache))
    q64 = q.double().to(dev).view(B, T, H, G, D)
    n, c = ints(lengths, dev)[:, None, None], ints([T] * B if counts is None else counts, dev)[:, None, None]
    j, t = torch.arange(192, device=dev)[None, None], torch.arange(T, device=dev)[None, :, None]
    inside = (j >= n) & (j - n < c)
    if masks is not None:
        inside = inside & ((masks.to(dev)[:, :, None] >> (j - n).clamp(0, 63)) & 1).bool()
    elif block == "causal":
        inside = inside & (j - n <= t)
    seen = ((j < n) | inside) & (t < c)
    for b in range(B):
        x = torch.einsum("thgd,hjd->thgj", q64[b], K[b]) * D ** -0.5
        mass = torch.einsum("thgd,hjd->thgj", q64[b].abs(), K[b].abs()) * D ** -0.5
        mass = mass.masked_fill(~seen[b][:, None, None], 0).amax(-1)
        x = x.masked_fill(~seen[b][:, None, None], float("-inf"))
        rl = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(rl > float("-inf"), rl, torch.zeros_like(rl))[..., None])
        ro = torch.einsum("thgj,hjd->thgd", p, V[b])
        weight = torch.einsum("thgj,hjd->thgd", p, V[b].abs())
        err = mass * 2.0 ** -16 + (q64[b].abs().sum(-1) * D ** -0.5 * 2.0 ** -20 if dtype == "f16" else 0)
        assert torch.all((out[b].double().view(T, H, G, D) - ro).abs()
                         <= weight * (2.0 ** -8 * 1.01 + 2 * err[..., None]) + 1e-30), b
        got = lse[b].double().view(T, H, G)
        f = rl > float("-inf")
        assert torch.equal(f, got > float("-inf"))
        assert torch.all((got[f] - rl[f]).abs() <= err[f] + 2.0 ** -20 * (1 + rl[f].abs()))


def test_cache_of_no_pages(pkg, dev):
    say("no pages")
    cache = pkg.KV4Cache(torch.empty(0, 2, 4352, dtype=torch.uint8, device=dev),
                         torch.zeros(2, 3, dtype=torch.int32, device=dev), 64)
    n = ints([100, 0], dev)
    q, kv = (torch.randn(2, 3, h, 64, device=dev).to(torch.bfloat16) for h in (4, 2))
    pkg.kv4_append(cache, kv, kv, n)
    k, v = pkg.kv4_read(cache, n, 3)
    out, lse = pkg.kv4_attention(q, cache, n)
    w = torch.rand(2, 2, 192, device=dev)
    nw = pkg.kv4_weights(q, cache, n, lse, w)
    nl, ew, source = pkg.kv4_evict(cache, n, w, 10, 2)
    torch.cuda.synchronize()
    assert not k.any() and not v.any() and not out.any() and torch.all(lse == float("-inf"))
    assert torch.equal(nw[0, :, :100], w[0, :, :100]) and not nw[0, :, 100:].any() and not nw[1].any()
    assert nl.tolist() == [10, 0] and torch.all(source[1] == -1)
    assert torch.equal(ew[0, 0, :10], w[0, 0][source[0, 0].long()])


def test_attention_takes_strides_given_outputs_and_other_streams(pkg, dev):
    say("attention strides")
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
        o, l = pkg.kv4_attention(qv, cache, lengths, out=out[..., :D].transpose(1, 2), lse=lse)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    assert l is lse and o.data_ptr() == out.data_ptr()
    check_attention(cache, q, "bf16", "causal", [100, 30], None, None, D ** -0.5, o, l)
    assert torch.all(out[..., D:] == 7.0)


def test_lengths_and_pages_out_of_range(pkg, dev):
    """Lengths are clamped to the table, counts to the block; slots of entries that name no page are not seen."""
    say("attention out of range")
    B, T, HQ, H, D = 4, 2, 2, 1, 64
    cache = random_cache(pkg, dev, B, H, D, 3, 21)
    K, V = contents(cache)
    cache.block_table[2, 1] = -1
    cache.block_table[3] = 10 ** 6
    q = torch.randn(B, T, HQ, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    lengths = ints([-5, 10 ** 6, 150, 150], dev)
    out, lse = pkg.kv4_attention(q.to(dev), cache, lengths, block="none", counts=ints([9, 9, 9, -1], dev))
    k, v = pkg.kv4_read(cache, lengths, 2)
    w = pkg.kv4_weights(q.to(dev), cache, lengths, lse, torch.zeros(B, H, 192, device=dev), block="none")
    pkg.kv4_append(cache, torch.zeros(B, T, H, D, device=dev), torch.zeros(B, T, H, D, device=dev),
                   ints([192, 10 ** 6, 70, 0], dev))
    torch.cuda.synchronize()
    assert torch.all(out[0] == 0) and torch.all(lse[0] == float("-inf")) and torch.all(out[3] == 0)
    assert torch.all(k[3] == 0) and torch.all(v[1] == 0)
    for b, seen in ((1, list(range(192))), (2, list(range(64)) + list(range(128, 150)))):
        ro, rl, weight, mass = O.attention(q[b:b + 1].double().numpy(), K[b:b + 1][:, :, seen], V[b:b + 1][:, :, seen],
                                           [len(seen)], [T], "none", D ** -0.5)
        tol = weight[0] * (2.0 ** -8 * 1.01 + 2.0 ** -15 * mass[0][..., None])
        assert np.all(np.abs(out[b].double().cpu().numpy() - ro[0]) <= tol)
        assert np.allclose(lse[b].double().cpu().numpy(), rl[0], atol=1e-3)
        assert abs(float(w[b].sum()) - T * HQ) < 1e-2
        assert torch.all(w[b, 0, [j for j in range(192) if j not in seen]] == 0)
    assert torch.all(w[0] == 0) and torch.all(w[3] == 0)


# ---- weights ------------------------------------------------------------------------

@pytest.mark.parametrize("B,T,HQ,H,D,pages,dtype,block,lengths,counts", ATTENTION)
def test_weights_match_oracle(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts):
    say("weights", B, T, HQ, H, D, pages, dtype, block, lengths, counts)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts, seed=B * T)
    arg = block if masks is None else masks.to(dev)
    n, c = ints(lengths, dev), ints(counts, dev)
    _, lse = pkg.kv4_attention(q.to(dev), cache, n, block=arg, counts=c)
    count = [T] * B if counts is None else counts
    w = torch.rand(B, H, cache.slots, generator=torch.Generator().manual_seed(8)) * 3
    K, _ = contents(cache)
    scale = D ** -0.5
    for accepted in (None, [(x + 1) // 2 for x in count]):
        wd = w.to(dev)
        got = pkg.kv4_weights(q.to(dev), cache, n, lse, wd, ints(accepted, dev), block=arg, counts=c)
        torch.cuda.synchronize()
        ref, added, mass = O.weights(q.double().numpy(), K, lengths, count, count if accepted is None else accepted,
                                     block, scale, lse.double().cpu().numpy(), w.double().numpy(),
                                     None if masks is None else masks.numpy())
        err = mass[..., None] * 2.0 ** -16 + (np.abs(q.double().numpy()).sum(-1).max() * scale * 2.0 ** -20
                                              if dtype == "f16" else 0.0)
        tol = added * (err + 2.0 ** -18) + ref * 2.0 ** -20
        assert np.all(np.abs(got.double().cpu().numpy() - ref) <= tol)
        assert torch.equal(wd.cpu(), w)
        turned = lse.transpose(0, 2).contiguous().transpose(0, 2)          # any strides
        same = pkg.kv4_weights(q.to(dev), cache, n, turned, wd, ints(accepted, dev), block=arg, counts=c, out=wd)
        assert same is wd and torch.equal(wd, got)


# ---- eviction -----------------------------------------------------------------------

EVICT = [
    # B, H, D, pages, lengths, keep, recent, weights
    (1, 1, 64, 1, [1], 1, 0, "rand"),
    (3, 2, 128, 3, [0, 190, 65], 64, 10, "rand"),
    (2, 1, 64, 3, [192, 130], 129, 0, "rand"),
    (2, 2, 128, 2, [100, 128], 99, 99, "rand"),            # all that stay are recent
    (2, 2, 128, 2, [100, 128], 20, 50, "equal"),           # a budget below `recent`
    (1, 3, 64, 40, [2500], 1000, 30, "rand"),
    (1, 2, 64, 40, [2560], 700, 1, "ties"),                # few distinct weights
    (2, 1, 128, 2, [100, 128], 300, 5, "rand"),            # a budget past the table
    (1, 2, 64, 20, [1279], 401, 7, "odd"),                 # NaN, infinities, both zeros
]


@pytest.mark.parametrize("B,H,D,pages,lengths,keep,recent,kind", EVICT)
def test_evict_keeps_the_oracles_slots(pkg, dev, B, H, D, pages, lengths, keep, recent, kind):
    say("evict", B, H, D, pages, lengths, keep, recent, kind)
    cache = random_cache(pkg, dev, B, H, D, pages, 70 + keep)
    g = torch.Generator().manual_seed(keep)
    w = torch.exp(3 * torch.randn(B, H, cache.slots, generator=g))
    if kind == "equal":
        w[:] = 0.5
    elif kind == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    elif kind == "odd":
        pick = torch.randint(0, 6, w.shape, generator=g)
        for i, x in enumerate((float("nan"), float("inf"), float("-inf"), 0.0, -0.0)):
            w[pick == i] = x
    before = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), D)
    wd = w.to(dev)
    nl, nw, source = pkg.kv4_evict(cache, ints(lengths, dev), wd, keep, recent)
    torch.cuda.synchronize()
    after = O.unpack(cache.data.cpu().numpy(), cache.block_table.cpu().numpy(), D)
    assert nl.tolist() == [min(n, keep) for n in lengths] and torch.equal(wd.cpu().nan_to_num(7), w.nan_to_num(7))
    nw, source = nw.cpu().numpy(), source.cpu().numpy()
    for b, n in enumerate(lengths):
        m = min(n, keep)
        for h in range(H):
            ref = O.evict(w[b, h, :n].double().numpy(), n, keep, recent)
            assert np.array_equal(source[b, h], ref), (b, h)
            assert np.array_equal(nw[b, h, :m], w[b, h].numpy()[ref[:m]], equal_nan=True)
            assert np.all(nw[b, h, m:] == 0)
            for x, y in zip(after, before):
                assert np.array_equal(x[b, h, :m], y[b, h][ref[:m]])
                assert np.array_equal(x[b, h, keep:], y[b, h, keep:])


@pytest.mark.parametrize("n,keep,recent,kind", [(5100, 900, 40, "rand"), (4480, 4000, 0, "ties"),
                                                (17000, 5000, 300, "rand"), (33001, 16500, 16000, "ties")])
def test_evict_from_long_sequences(pkg, dev, n, keep, recent, kind):
    """More slots than one walk of the selection holds, with the budget inside and past the first."""
    say("evict long", n, keep, recent, kind)
    pages = -(-n // 64)
    data = torch.randint(0, 256, (pages, 1, 4352), generator=torch.Generator().manual_seed(n), dtype=torch.uint8)
    cache = pkg.KV4Cache(data.to(dev), torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)[None], 64)
    g = torch.Generator().manual_seed(keep)
    w = torch.exp(3 * torch.randn(1, 1, cache.slots, generator=g))
    if kind == "ties":
        w = torch.randint(0, 5, w.shape, generator=g).float()
    k0, v0 = pkg.kv4_read(cache, ints([0], dev), n, dtype=torch.float32)
    _, nw, source = pkg.kv4_evict(cache, ints([n], dev), w.to(dev), keep, recent)
    k1, v1 = pkg.kv4_read(cache, ints([0], dev), keep, dtype=torch.float32)
    torch.cuda.synchronize()
    ref = torch.tensor(O.evict(w[0, 0, :n].double().numpy(), n, keep, recent))
    assert torch.equal(source[0, 0].cpu().long(), ref)
    assert torch.equal(nw[0, 0, :keep].cpu(), w[0, 0][ref]) and not nw[0, 0, keep:].any()
    for a, b in ((k0, k1), (v0, v1)):
        assert torch.equal(a[0, ref.to(dev)].view(torch.int32), b[0].view(torch.int32))


# ---- together -------------------------------------------------------------------------

def test_calls_replay_in_a_graph(pkg, dev):
    """Append, attention, weights and eviction captured once and replayed on new inputs and lengths."""
    say("graph")
    B, T, HQ, H, D, S = 2, 4, 4, 2, 64, 512
    caches = [pkg.KV4Cache.allocate(B, S, H, D, dev) for _ in range(2)]
    g = torch.Generator(device=dev).manual_seed(4)
    q = torch.empty(B, T, HQ, D, dtype=torch.bfloat16, device=dev)
    k, v = (torch.empty(B, T, H, D, dtype=torch.bfloat16, device=dev) for _ in "kv")
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    w = torch.zeros(B, H, S, device=dev)

    def step(cache, lengths, w):
        pkg.kv4_append(cache, k, v, lengths)
        out, lse = pkg.kv4_attention(q, cache, lengths)
        w2 = pkg.kv4_weights(q, cache, lengths, lse, w)
        nl, nw, _ = pkg.kv4_evict(cache, lengths + T, w2, 40, 8)
        return out, lse, nl, nw

    def fill():
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))

    fill()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(caches[0], lengths, w)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    caches[0].data.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0], lengths, w)
        lengths.copy_(captured[2])
        w.copy_(captured[3])
    el, ew = torch.zeros_like(lengths), torch.zeros_like(w)
    lengths.zero_()
    w.zero_()
    for i in range(16):                                    # past the budget from the eleventh on
        fill()
        graph.replay()
        torch.cuda.synchronize()
        eager = step(caches[1], el, ew)
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), i
        el, ew = eager[2], eager[3]
    assert el.tolist() == [40, 40] and torch.equal(caches[0].data, caches[1].data)


def test_repeated_calls_are_bit_identical(pkg, dev):
    say("repeat")
    cache, q, _ = attention_inputs(pkg, dev, 3, 16, 8, 2, 128, 20, "bf16", "causal", [1200, 700, 3], None, 31)
    lengths, qd = ints([1200, 700, 3], dev), q.to(dev)
    w = torch.rand(3, 2, cache.slots, device=dev)
    first = pkg.kv4_attention(qd, cache, lengths)
    fw = pkg.kv4_weights(qd, cache, lengths, first[1], w)
    for _ in range(5):
        o, l = pkg.kv4_attention(qd, cache, lengths)
        assert torch.equal(o, first[0]) and torch.equal(l, first[1])
        assert torch.equal(pkg.kv4_weights(qd, cache, lengths, l, w), fw)


def test_refusals(pkg, dev):
    cache = pkg.KV4Cache.allocate(2, 100, 2, 64, dev)
    assert cache.slots == 128
    bf = torch.bfloat16
    q = torch.zeros(2, 3, 4, 64, dtype=bf, device=dev)
    kv = torch.zeros(2, 3, 2, 64, dtype=bf, device=dev)
    n = ints([0, 0], dev)
    lse, w = torch.zeros(2, 3, 4, device=dev), torch.zeros(2, 2, 128, device=dev)
    with pytest.raises(ValueError, match="head_dim must be one of"):
        pkg.KV4Cache.allocate(1, 64, 1, 80, dev)
    with pytest.raises(ValueError, match="data must be uint8"):
        pkg.KV4Cache(cache.data[..., :-1], cache.block_table, 64)
    with pytest.raises(ValueError, match="data must be contiguous"):
        pkg.KV4Cache(cache.data[::2], cache.block_table, 64)
    with pytest.raises(ValueError, match="block_table must be int32"):
        pkg.KV4Cache(cache.data, cache.block_table.long(), 64)
    with pytest.raises(ValueError, match="no CPU fallback"):
        pkg.kv4_append(cache, kv.cpu(), kv, n)
    with pytest.raises(ValueError, match="one shape and dtype"):
        pkg.kv4_append(cache, kv, kv.float(), n)
    with pytest.raises(ValueError, match=r"k must be \[2, T, 2, 64\]"):
        pkg.kv4_append(cache, q, q, n)
    with pytest.raises(ValueError, match="lengths must be int32"):
        pkg.kv4_append(cache, kv, kv, n.long())
    with pytest.raises(ValueError, match="unit channel stride"):
        pkg.kv4_append(cache, kv.transpose(2, 3).contiguous().transpose(2, 3), kv, n)
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        odd = torch.zeros(2, 3, 2, 67, dtype=bf, device=dev)[..., :64]
        pkg.kv4_append(cache, odd, odd, n)
    with pytest.raises(TypeError, match="q dtype"):
        pkg.kv4_attention(q.float(), cache, n)
    with pytest.raises(ValueError, match="do not divide"):
        pkg.kv4_attention(q[:, :, :3], cache, n)
    with pytest.raises(ValueError, match="block must be one of"):
        pkg.kv4_attention(q, cache, n, block="window")
    with pytest.raises(ValueError, match="block mask must be int64"):
        pkg.kv4_attention(q, cache, n, block=torch.zeros(2, 2, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="holds 64 slots"):
        pkg.kv4_attention(torch.zeros(2, 65, 4, 64, dtype=bf, device=dev), cache, n,
                          block=torch.zeros(2, 65, dtype=torch.int64, device=dev))
    with pytest.raises(RuntimeError, match="scale must be finite"):
        pkg.kv4_attention(q, cache, n, scale=float("nan"))
    with pytest.raises(ValueError, match="out must be"):
        pkg.kv4_attention(q, cache, n, out=q[:, :1])
    with pytest.raises(ValueError, match="lse must be"):
        pkg.kv4_weights(q, cache, n, lse[:, :1], w)
    with pytest.raises(ValueError, match="weights must be"):
        pkg.kv4_weights(q, cache, n, lse, w[..., :100])
    with pytest.raises(ValueError, match="keep must be"):
        pkg.kv4_evict(cache, n, w, 0)
    # an empty block is nothing to do
    pkg.kv4_append(cache, kv[:, :0], kv[:, :0], n)
    o, l = pkg.kv4_attention(q[:, :0], cache, n)
    assert o.shape == (2, 0, 4, 64) and l.shape == (2, 0, 4)
