"""CPU tests of the bound that attention's outputs are held to: it holds for weights in two
bf16 parts, and a mistake of one part's size (planted in a restatement of the sums) passes it
nowhere."""

import numpy as np
import pytest

from oracle import kv4 as O


def sums(p, codes, scale, parts, dtype):
    """Outputs of one row from weights p [n], value codes [n, D] and scales [n], in the kernel's roundings."""
    w = (p * scale).astype(np.float32)
    hi = O.round_to(w, "bf16")
    total = hi @ codes
    if parts == 2:
        total = total + O.round_to(w - hi.astype(np.float32), "bf16") @ codes
    return O.round_to(total / p.astype(np.float64).sum(), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 5, 40, 200])
def test_one_part_of_the_weights_is_outside(n, dtype):
    rng = np.random.default_rng(n)
    D, rows, outside = 64, 60, {1: 0, 2: 0}
    for _ in range(rows):
        x = rng.normal(size=n)
        p = np.exp(x - x.max()).astype(np.float32)
        codes = O.decode(rng.integers(0, 16, size=(n, D)).astype(np.uint8))
        scale = O.round_to(rng.uniform(0.1, 1.1, size=n), "bf16").astype(np.float32)
        exact = np.exp(x - x.max())
        V = codes * scale[:, None]
        out, weight = exact @ V / exact.sum(), exact @ np.abs(V) / exact.sum()
        lo, hi = O.output_range(out[None], weight[None], np.array([0.0]), dtype)
        for parts in (1, 2):
            got = sums(p, codes, scale, parts, dtype)
            outside[parts] += int(np.any((got < lo[0]) | (got > hi[0])))
    assert outside[2] == 0
    if n > 1:                                      # of one slot the weight cancels but for its rounding with the scale
        assert outside[1] > rows // 2


def test_range_is_one_number_or_two_where_nothing_is_off():
    x = np.array([[1.0, -0.3, 1e-3, 2.5e4]])
    for dtype in ("bf16", "f16"):
        lo, hi = O.output_range(x, np.abs(x), np.zeros(1), dtype)
        r = O.round_to(x, dtype)
        assert np.all(lo <= r) and np.all(r <= hi)
        assert np.all(hi - lo <= np.abs(x) * 2.0 ** -6)
