"""CPU restatement of the 4-bit key/value cache, in numpy and 64 bits.

Format, rounding and the five operations as include/dels.h defines them; slow and
plain on purpose.  Lengths and counts here are within range (the kernels' clamping
is tested by itself).
"""

from __future__ import annotations

import numpy as np

PAGE = 64
LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
MIDPOINTS = (LEVELS[1:] + LEVELS[:-1]) / 2
BIG = 3.0e38


def page_bytes(D: int) -> int:
    return 66 * D + 128


def _clean(x):
    x = np.asarray(x, dtype=np.float64)
    return np.clip(np.where(np.isnan(x), 0.0, x), -np.float64(np.float32(BIG)), np.float64(np.float32(BIG)))


def encode(y):
    """Codes of y = x / scale: nearest level, ties to the even code, sign bit for y < 0."""
    a = np.abs(y)
    code = np.zeros(a.shape, dtype=np.uint8)
    for i, mid in enumerate(MIDPOINTS):
        up = a > mid if i % 2 == 0 else a >= mid      # between codes i and i + 1: a tie goes to the even one
        code[up] = i + 1
    return code | np.where(y < 0, 8, 0).astype(np.uint8)


def decode(codes):
    return np.where(codes & 8, -1.0, 1.0) * LEVELS[codes & 7]


def encode_keys(k):
    """(codes, exponent bytes) of keys [..., D]."""
    x = _clean(k)
    x = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(x).max(-1)
    e = np.full(amax.shape, 1, dtype=np.int64)
    for step in range(1, 252):                        # the smallest exponent whose sevenfold holds amax
        e = np.where(7.0 * 2.0 ** (step - 127) < amax, step + 1, e)
    return encode(x / 2.0 ** (e[..., None] - 127)).reshape(*x.shape[:-2], -1), e.astype(np.uint8)


def _bf16(x):
    """float32 -> nearest bf16 (ties to even), as float64."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32).astype(np.float64)


def encode_values(v):
    """(codes, scales) of values [..., D]."""
    x = _clean(v)
    amax = np.abs(x).max(-1).astype(np.float32)
    scale = np.maximum(_bf16(amax * np.float32(1.0 / 6.0)), 2.0 ** -126)
    return encode(x / scale[..., None]), scale


def key_values(codes, e):
    y = decode(codes)
    y = y.reshape(*y.shape[:-1], -1, 32) * 2.0 ** (e.astype(np.float64)[..., None] - 127)
    return y.reshape(*codes.shape)


def value_values(codes, scale):
    return decode(codes) * scale[..., None]


def unpack_page(page, D):
    """(key codes [64, D], exponents [64, D/32], value codes [64, D], value scales [64]) of one page's bytes."""
    kc = np.empty((PAGE, D), np.uint8)
    ke = np.empty((PAGE, D // 32), np.uint8)
    vc = np.empty((PAGE, D), np.uint8)
    vs = np.empty(PAGE, np.float64)
    words = page[34 * D:66 * D].view("<u4").reshape(8, D)
    scales = page[66 * D:].view("<u2").astype(np.uint32) << 16
    for j in range(PAGE):
        row = page[j * D // 2:(j + 1) * D // 2]
        kc[j, 0::2], kc[j, 1::2] = row & 15, row >> 4
        for m in range(D // 32):
            ke[j, m] = page[32 * D + 64 * m + 16 * (j >> 3 & 3) + 4 * (j & 3) + 2 * (j >> 5) + (j >> 2 & 1)]
        vc[j] = (words[j >> 3] >> np.uint32(4 * (j & 7))) & 15
        vs[j] = scales[j:j + 1].view(np.float32)[0]
    return kc, ke, vc, vs


def unpack(data, table, D):
    """Codes and scales of every slot, [B, H, slots, ...], of pages [N, H, bytes] and a valid table."""
    out = []
    for row in table:
        heads = []
        for h in range(data.shape[1]):
            pages = [unpack_page(data[p, h], D) for p in row]
            heads.append([np.concatenate(x) for x in zip(*pages)])
        out.append([np.stack(x) for x in zip(*heads)])
    return [np.stack(x) for x in zip(*out)]


def sees(j, n, count, t, block, bits):
    i = j - n
    if i < 0:
        return True
    if i >= count or block == "none":
        return False
    if block == "causal":
        return i <= t
    return True if block == "full" else bool((int(bits) >> i) & 1)


def _scores(q, K, h, t, n, count, block, bits, scale):
    """Scores of one (row, head) over all slots, -inf where unseen; the largest sum of |q k| * |scale|; which are seen."""
    vis = np.array([sees(j, n, count, t, block, bits) for j in range(K.shape[0])], dtype=bool)
    x = np.where(vis, scale * (K @ q), -np.inf)
    mass = (np.abs(K) @ np.abs(q))[vis].max() * abs(scale) if vis.any() else 0.0
    return x, mass, vis


def attention(q, K, V, lengths, counts, block, scale, masks=None):
    """q [B, T, HQ, D]; K, V [B, H, slots, D].  Returns out, lse, and for bounds: sum p |v| / sum p, the mass."""
    B, T, HQ, D = q.shape
    H = K.shape[1]
    out, lse = np.zeros((B, T, HQ, D)), np.full((B, T, HQ), -np.inf)
    weight, mass = np.zeros((B, T, HQ, D)), np.zeros((B, T, HQ))
    for b in range(B):
        for t in range(int(counts[b])):
            for hq in range(HQ):
                h = hq // (HQ // H)
                x, mass[b, t, hq], _ = _scores(q[b, t, hq], K[b, h], h, t, lengths[b], counts[b], block,
                                               masks[b, t] if masks is not None else 0, scale)
                if np.all(x == -np.inf):
                    continue
                p = np.exp(x - x.max())
                out[b, t, hq] = p @ V[b, h] / p.sum()
                weight[b, t, hq] = p @ np.abs(V[b, h]) / p.sum()
                lse[b, t, hq] = x.max() + np.log(p.sum())
    return out, lse, weight, mass


def weights(q, K, lengths, counts, accepted, block, scale, lse, w, masks=None):
    """The new weights [B, H, slots], the sums that were added, and the largest mass of their rows."""
    B, T, HQ, D = q.shape
    H = K.shape[1]
    old = np.array(w, dtype=np.float64)
    added, mass = np.zeros_like(old), np.zeros(old.shape[:2])
    for b in range(B):
        old[b, :, lengths[b]:] = 0
        for t in range(min(int(accepted[b]), int(counts[b]))):
            for hq in range(HQ):
                if lse[b, t, hq] == -np.inf:
                    continue
                h = hq // (HQ // H)
                x, m, vis = _scores(q[b, t, hq], K[b, h], h, t, lengths[b], counts[b], block,
                                    masks[b, t] if masks is not None else 0, scale)
                added[b, h] += np.where(vis, np.exp(x - lse[b, t, hq]), 0.0)
                mass[b, h] = max(mass[b, h], m)
    return old + added, added, mass


def evict(w, n, keep, recent, named=None):
    """Sources [keep] of one (sequence, head) of n slots with weights w; named: whether each lies in a page."""
    if n <= keep:
        return np.array(list(range(n)) + [-1] * (keep - n))
    named = np.ones(n, dtype=bool) if named is None else named
    room = int(named[:keep].sum())
    recent = min(recent, room)
    clean = np.where(np.isnan(w), -np.inf, w)
    stay = {j for j in range(n - recent, n) if named[j]}
    order = sorted((j for j in range(n - recent) if named[j]), key=lambda j: (-clean[j], j))
    stay |= set(order[:room - len(stay)])
    holes = [j for j in range(keep) if named[j] and j not in stay]
    movers = sorted(j for j in stay if j >= keep)
    source = np.arange(keep)
    source[holes] = movers
    return source


def round_to(x, dtype):
    """Nearest number of a type ("bf16", "f16"), as float64."""
    if dtype == "bf16":
        return _bf16(x)
    with np.errstate(over="ignore"):
        return np.asarray(x, dtype=np.float64).astype(np.float16).astype(np.float64)


def output_range(out, weight, err, dtype):
    """The numbers of a type that attention's outputs may be: (lowest, highest).

    err [B, T, HQ]: how far a row's scores may be off.  The weights then are off by that, by
    the 2^-20 of an argument of the exponential around the row's largest score, and by the
    two bf16 parts that meet the values (2^-17); sums in fp32 over a few hundred slots add
    as much.  What comes of it is rounded once, to its type: whatever lies between the
    roundings of both ends is right.
    """
    off = weight * (2.0 ** -16 + 2.0 * (err[..., None] + 2.0 ** -20)) + 1e-30
    return round_to(out - off, dtype), round_to(out + off, dtype)
