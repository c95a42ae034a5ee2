"""CPU restatement of the 8-bit key/value cache, in numpy and 64 bits.

Format, rounding, rotation and the three operations as include/dels.h defines them; slow
and plain on purpose.  Lengths and counts here are within range (the kernels' clamping is
tested by itself).
"""

from __future__ import annotations

import numpy as np

from . import kv4

PAGE, BLOCK = 64, 32
LOW, HIGH = 63, 191
MOST = 448.0 * 2.0 ** 64
# magnitudes of the codes 0 .. 126, and the middles between neighbours
LEVELS = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                   for e in range(16) for m in range(8)][:127])
MIDDLES = (LEVELS[1:] + LEVELS[:-1]) / 2


def page_bytes(D: int) -> int:
    return 128 * D + 128


def place(s: int) -> int:
    """Where a block's keys have its slot s."""
    return 8 * (s % 16 // 4) + 4 * (s // 16) + s % 4


def encode(y):
    """Codes of |y| <= 448: nearest level, ties to the even code, sign bit for y < 0 (and -0)."""
    a = np.abs(y)
    code = np.searchsorted(MIDDLES, a, side="left")            # middles below a
    tie = (code < 126) & (MIDDLES[np.minimum(code, 125)] == a)
    code = code + (tie & (code % 2 == 1))
    return (code + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def decode(codes):
    x = np.append(LEVELS, np.nan)[codes & 127]
    return np.where(codes & 128, -x, x)


def exponent(top):
    """The smallest of LOW .. HIGH whose power of two holds `top` 448-fold."""
    for e in range(LOW, HIGH):
        if 448.0 * 2.0 ** (e - 127) >= top:
            return e
    return HIGH


def unpack(data, table, D):
    """What the slots of pages [N, H, bytes] and a valid table hold.

    kc, vc codes [B, H, slots, D]; ke, ve exponents [B, H, slots / 32]; bad [B, H, slots].
    """
    B, P = table.shape
    H = data.shape[1]
    kc, vc = (np.empty((B, H, P * PAGE, D), np.uint8) for _ in "kv")
    ke, ve = (np.empty((B, H, P * 2), np.uint8) for _ in "kv")
    bad = np.empty((B, H, P * PAGE), bool)
    slots = np.arange(PAGE)
    u, s = slots // BLOCK, slots % BLOCK
    pos = np.array([place(int(i)) for i in s])
    c = np.arange(D)
    kat = (32 * D * u + 16 * pos)[:, None] + 512 * (c // 16) + c % 16
    vat = (64 * D + 32 * D * u + 16 * D * (s // 16) + s % 16)[:, None] + 16 * c
    for b in range(B):
        for p in range(P):
            page = data[table[b, p]]
            at = slice(p * PAGE, (p + 1) * PAGE)
            kc[b, :, at], vc[b, :, at] = page[:, kat], page[:, vat]
            head = page[:, 128 * D:128 * D + 16].reshape(H, 2, 8)
            ke[b, :, 2 * p:2 * p + 2], ve[b, :, 2 * p:2 * p + 2] = head[..., 0], head[..., 1]
            words = np.ascontiguousarray(head[..., 4:]).view("<u4")[..., 0]
            bad[b, :, at] = (words[:, u] >> s) & 1
    return kc, ke, vc, ve, bad


def values(codes, e, bad):
    """Numbers [B, H, slots, D] of codes and exponents; NaN where a row was not finite."""
    x = decode(codes) * np.repeat(2.0 ** (e.astype(np.float64) - 127), BLOCK, 2)[..., None]
    return np.where(bad[..., None], np.nan, x)


def rotate(x, cos, sin, at, interleaved):
    """Rows [..., D] of float32 rotated by the angles of positions `at` [...]; NaN where there are none."""
    x = np.array(x, dtype=np.float32)
    half = cos.shape[1]
    i = np.arange(half)
    i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    have = (at >= 0) & (at < cos.shape[0])
    row = np.where(have, at, 0)
    c, s = cos[row].astype(np.float32), sin[row].astype(np.float32)
    a, b = x[..., i].copy(), x[..., j].copy()
    with np.errstate(invalid="ignore", over="ignore"):
        x[..., i] = np.where(have[..., None], a * c - b * s, np.nan)
        x[..., j] = np.where(have[..., None], b * c + a * s, np.nan)
    return x


def append(state, k, v, n, count):
    """Changes an unpacked cache (of one sequence: arrays [H, ...]) as the call does for rows k, v [T, H, D] at n."""
    kc, ke, vc, ve, bad = state
    H, slots = kc.shape[:2]
    end = min(n + count, slots)
    if end <= n:
        return
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    with np.errstate(invalid="ignore"):
        none = ~((np.abs(k) <= MOST).all(-1) & (np.abs(v) <= MOST).all(-1))      # [T, H]
    for first in range(n // BLOCK * BLOCK, end, BLOCK):
        lo, hi, u = max(first, n), min(first + BLOCK, end), first // BLOCK
        for h in range(H):
            bad[h, lo:hi] = none[lo - n:hi - n, h]
            bad[h, hi:first + BLOCK] = False
            for codes, exps, x in ((kc, ke, k), (vc, ve, v)):
                rows = np.where(none[lo - n:hi - n, h, None], 0.0, x[lo - n:hi - n, h])
                e = exponent(np.abs(rows).max())
                if lo > first:
                    was = min(max(int(exps[h, u]), LOW), HIGH)
                    if e > was:
                        codes[h, first:lo] = encode(decode(codes[h, first:lo]) * 2.0 ** (was - e))
                    e = max(e, was)
                exps[h, u] = e
                codes[h, lo:hi] = encode(rows * 2.0 ** (127 - e))


def visible(n, count, T, slots, block, masks=None, window=None, sinks=0, positions=None):
    """Which slots the rows of a block see, [T, slots]; the window goes by slots or by the rows' positions [T]."""
    j, t = np.arange(slots)[None], np.arange(T)[:, None]
    i = j - n
    if masks is not None:
        own = ((masks[:, None].astype(np.uint64) >> np.clip(i, 0, 63).astype(np.uint64)) & np.uint64(1)).astype(bool)
    else:
        own = {"causal": i <= t, "full": i >= 0, "none": np.zeros((T, slots), bool)}[block]
    see = (i < 0) | (own & (i < count))
    if window is not None and positions is not None:
        depth = np.clip(np.asarray(positions, np.int64) - n, 0, T - 1)
        place = np.where((i >= 0) & (i < T), depth[np.clip(i, 0, T - 1)], i)
        see = see & ((place > depth[:, None] - window) | (n + place < sinks))
    elif window is not None:
        see = see & ((i > t - window) | (j < sinks))
    return see & (t < count)


def attention(q, K, V, lengths, counts, block, scale, masks=None, window=None, sinks=0, positions=None):
    """q [B, T, HQ, D]; K, V [B, H, slots, D] (NaN: not finite).

    Returns out, lse, and for bounds: sum p |v| / sum p, and the largest sum of |q k| * |scale|
    over the slots that a row sees.  A row that sees a NaN is NaN.
    """
    B, T, HQ, D = q.shape
    H, slots = K.shape[1:3]
    G = HQ // H
    out, lse = np.zeros((B, T, HQ, D)), np.full((B, T, HQ), -np.inf)
    weight, mass = np.zeros((B, T, HQ, D)), np.zeros((B, T, HQ))
    for b in range(B):
        see = visible(lengths[b], counts[b], T, slots, block, None if masks is None else masks[b], window, sinks,
                      None if positions is None else positions[b])
        for h in range(H):
            none = np.isnan(K[b, h]).any(-1)
            k, v = np.nan_to_num(K[b, h]), np.nan_to_num(V[b, h])
            for hq in range(h * G, (h + 1) * G):
                x = np.where(see, scale * (q[b, :, hq] @ k.T), -np.inf)
                big = np.where(see, abs(scale) * (np.abs(q[b, :, hq]) @ np.abs(k).T), 0.0)
                mass[b, :, hq] = big.max(-1, initial=0.0)
                top = x.max(-1, initial=-np.inf)
                some = top > -np.inf
                p = np.exp(x - np.where(some, top, 0.0)[:, None])
                total = p.sum(-1)
                safe = np.where(some, total, 1.0)
                out[b, :, hq] = np.where(some[:, None], p @ v / safe[:, None], 0.0)
                weight[b, :, hq] = p @ np.abs(v) / safe[:, None]
                lse[b, :, hq] = np.where(some, top + np.log(safe), -np.inf)
                lost = (see & none[None]).any(-1)
                out[b, lost, hq], lse[b, lost, hq] = np.nan, np.nan
    return out, lse, weight, mass


def output_range(out, weight, err, dtype, most, parts=1):
    """The numbers of a type that attention's outputs may be: (lowest, highest).

    err [B, T, HQ]: how far a row's scores may be off.  The weights then are off by that, by
    the 2^-20 of an argument of the exponential around the row's largest score, and by the f16
    number, or two of them for f16 outputs, that meets the values: 2^-11 or 2^-22 of each weight, and
    2^-32 of the row's largest where that is more (`most`: slots times the largest |value|).  A block
    whose scale is far below the largest takes two bf16 parts, 2^-17, as all do where a bf16 output is
    asked for with weights in two `parts`.  Sums in fp32 over a few
    hundred slots add 2^-16.  What comes of it is rounded once, to its type: whatever lies
    between the roundings of both ends is right.
    """
    part = 2.0 ** -11 if dtype == "bf16" and parts == 1 else 2.0 ** -17
    off = weight * (part + 2.0 ** -16 + 2.0 * (err[..., None] + 2.0 ** -20)) + most * 2.0 ** -32 + 1e-30
    return kv4.round_to(out - off, dtype), kv4.round_to(out + off, dtype)
