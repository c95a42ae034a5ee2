"""GPU tests of rows that enter a block whose kept rows are smaller by up to 2^128.

A block's exponents are 63 .. 191, so a new row may raise one by any number up to 128: kept codes are
then rounded under a power of two of 2^-128 .. 2^-1, of which those below 2^-18 leave zeros of
their sign.  What append writes is compared with the oracle to the byte.
"""

import numpy as np
import pytest
import torch

from oracle import kv8 as O
from test_gpu_kv8 import NAN, ints, say, unpacked

pytestmark = pytest.mark.gpu

H = 2


def first_rows(kind, n, D, g):
    """Rows [1, n, H, D] that leave a block at exponent 63: nothing, next to nothing, codes of all sizes, none held."""
    sign = torch.where(torch.rand(1, n, H, D, generator=g) < 0.5, -1.0, 1.0)
    if kind == "zeros":
        return sign * 0.0
    if kind == "tiny":
        return sign * 2.0 ** -70
    if kind == "codes":
        x = sign * torch.exp2(-18 * torch.rand(1, n, H, D, generator=g)) * 448.0 * 2.0 ** -64
        x[..., 0] = 448.0 * 2.0 ** -64
        return x
    return torch.full((1, n, H, D), NAN)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["zeros", "tiny", "codes", "not held"])
@pytest.mark.parametrize("steps", [[64], [63], [62], [61, 64], [-63, -62, 63, 64], [-46, 0, 46, 64]])
@pytest.mark.parametrize("first", [0, 32, 69])
def test_kept_rows_under_much_larger_exponents(pkg, dev, D, kind, steps, first):
    """Rows of 448 * 2^e in calls of their own; values take the steps that keys do, the other way round, or none."""
    say("jump", D, kind, steps, first)
    g = torch.Generator().manual_seed(D + first)
    for way in ("both", "keys", "values", "turned"):
        cache = pkg.KV8Cache.allocate(1, 128, H, D, dev)
        state = [x[0] for x in unpacked(cache)]
        at = first

        def put(k, v):
            nonlocal at
            pkg.kv8_append(cache, k.to(dev), v.to(dev), ints([at], dev))
            O.append(state, k[0].numpy(), v[0].numpy(), at, k.shape[1])
            at += k.shape[1]
            torch.cuda.synchronize()
            for got, want in zip(unpacked(cache), state):
                assert np.array_equal(got[0], want), (way, at)

        put(first_rows(kind, 7, D, g), first_rows(kind, 7, D, g))
        small = 2.0 ** -71 * torch.randn(1, 3, H, D, generator=g)
        for i, e in enumerate(steps):
            big = torch.randn(1, 3, H, D, generator=g).clamp(-1, 1) * 448.0 * 2.0 ** e
            big[0, 1, :, 5] = 448.0 * 2.0 ** e
            back = torch.randn(1, 3, H, D, generator=g).clamp(-1, 1) * 448.0 * 2.0 ** steps[-1 - i]
            put(big if way != "values" else small, {"both": -big, "keys": small, "values": big, "turned": back}[way])


@pytest.mark.parametrize("old", range(63, 192, 16))
def test_every_pair_of_exponents(pkg, dev, old):
    """A block of every exponent from `old` on, and a row of every larger one behind it."""
    say("pairs", old)
    D = 64
    pairs = [(o, e) for o in range(old, min(old + 16, 192)) for e in range(o, 192, 1 if o == 63 else 5)]
    pairs += [(o, 191) for o in range(old, min(old + 16, 192))]
    g = torch.Generator().manual_seed(old)
    cache = pkg.KV8Cache.allocate(len(pairs), 32, 1, D, dev)
    o, e = (torch.tensor(x).double() - 127 for x in zip(*pairs))
    k = torch.randn(len(pairs), 6, 1, D, generator=g, dtype=torch.float64).clamp(-1, 1) * 448
    k[:, :, :, 9], k[:, :, :, 10] = 448, -448
    k[:, :4] *= torch.exp2(o)[:, None, None, None]
    k[:, 4:] *= torch.exp2(e)[:, None, None, None]
    k = k.float()
    v = -k.flip(-1)
    zero = [0] * len(pairs)
    pkg.kv8_append(cache, k[:, :4].to(dev), v[:, :4].to(dev), ints(zero, dev))
    pkg.kv8_append(cache, k[:, 4:].to(dev), v[:, 4:].to(dev), ints([4] * len(pairs), dev))
    torch.cuda.synchronize()
    got = unpacked(cache)
    for b, pair in enumerate(pairs):
        state = [np.zeros_like(x[b]) for x in got]
        O.append(state, k[b, :4].numpy(), v[b, :4].numpy(), 0, 4)
        assert state[1][0, 0] == state[3][0, 0] == pair[0]
        O.append(state, k[b, 4:].numpy(), v[b, 4:].numpy(), 4, 2)
        for x, want in zip(got, state):
            assert np.array_equal(x[b], want), pair
