"""CPU tests of the bound of weights in two parts, and of the argument that asks for them.

A weight in one f16 number, planted in a restatement of the sums, lies outside of the bound where values cancel
and, with small scores, in ordinary sums; two bf16 or two f16 numbers never do.
"""

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv4, kv8 as O
from test_kv8_host import cache, on_cpu, small  # noqa: F401


def sums(p, v, parts, kind):
    """One row from weights p [n] relative to their largest and values v [n, D], as the kernel rounds them."""
    w = (p * 2.0 ** 7).astype(np.float32)                 # up to 2^7 .. 2^15
    hi = kv4.round_to(w, kind)
    total = hi @ v
    if parts == 2:
        total = total + kv4.round_to(w - hi.astype(np.float32), kind) @ v
    return kv4.round_to(total / w.astype(np.float64).sum(), "bf16")


@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("n", [2, 10, 300])
def test_one_part_is_outside(n, cancel):
    rng = np.random.default_rng(n)
    D, rows = 128, 40
    out_of = dict(one=0, two_f16=0, two_bf16=0)
    for _ in range(rows):
        x = rng.normal(size=n) * 0.3
        exact = np.exp(x - x.max())
        v = O.LEVELS[rng.integers(40, 90, size=(n, D))] * rng.choice([-1.0, 1.0], size=(n, D))
        if cancel:
            v[1::2] = -v[:n - 1:2]
        out, weight = exact @ v / exact.sum(), exact @ np.abs(v) / exact.sum()
        lo, hi = O.output_range(out[None], weight[None], np.zeros(1), "bf16", 0.0, 2)
        p = exact.astype(np.float32)
        for name, parts, kind in (("one", 1, "f16"), ("two_f16", 2, "f16"), ("two_bf16", 2, "bf16")):
            got = sums(p, v, parts, kind)
            out_of[name] += int(np.any((got < lo[0]) | (got > hi[0])))
        one_lo, one_hi = O.output_range(out[None], weight[None], np.zeros(1), "bf16", 0.0)
        got = sums(p, v, 1, "f16")
        assert np.all((got >= one_lo[0]) & (got <= one_hi[0]))
    # two parts nowhere; one part in some row at least (of two slots one ratio makes all channels, whose
    # values have eight different mantissas: few outputs lie near a border of the bound)
    assert out_of["two_f16"] == out_of["two_bf16"] == 0 and out_of["one"] > 0, out_of


def test_refusals_before_the_gpu(pkg):
    lib = pkg._lib.load()

    def attention(parts):
        ref = ctypes.byref(pkg._lib.Kv8OptionsParams(None, 0, parts))
        return lib.dels_kv8_attention_ex(cache(pkg), 0x1000, 4096, 1024, 128, 1, 8, 4, 0x3000, None, 0, None, 0, 1.0,
                                         0, 0, ref, 0x4000, 4096, 1024, 128, 0x5000, 0x6000, 16, None)

    assert attention(0) == attention(1) == attention(2) == -4      # all checks passed but the workspace's
    for parts in (-1, 3):
        assert attention(parts) == -1 and b"parts" in lib.dels_last_error()


def test_weight_parts_argument(on_cpu):  # noqa: F811
    pkg, got = on_cpu
    lib, calls = pkg.kv8._lib.load(), []
    lib.dels_kv8_attention_ex = lambda *a: calls.append(a) or 0
    c, n = small(pkg), torch.zeros(2, dtype=torch.int32)
    q, ws = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(1 << 18, dtype=torch.uint8)
    for parts in (0, 3, None, "2"):
        with pytest.raises(ValueError, match="weight_parts must be 1 or 2"):
            pkg.kv8_attention(q, c, n, workspace=ws, weight_parts=parts)
    pkg.kv8_attention(q, c, n, workspace=ws, weight_parts=1)
    assert len(got) == 1 and not calls
    pkg.kv8_attention(q, c, n, workspace=ws, weight_parts=2)
    options = calls[-1][16]._obj
    assert len(got) == 1 and (options.positions, options.ld_positions, options.weight_parts) == (None, 0, 2)
