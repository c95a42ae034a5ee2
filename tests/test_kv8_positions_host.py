"""CPU tests of windows over trees: the oracle's visibility by positions, and the call's argument checks."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv8 as O
from test_kv8_host import cache, on_cpu, small  # noqa: F401


def test_a_rows_window_is_that_of_its_branch():
    """Context slots and ancestors within the window of a row's position, sinks by position."""
    rng = np.random.default_rng(1)
    for _ in range(200):
        T, n, window, sinks = (int(rng.integers(*r)) for r in ((1, 20), (0, 30), (1, 25), (0, 40)))
        parent = [int(rng.integers(-1, t)) if t else -1 for t in range(T)]
        paths = []
        for t in range(T):
            paths.append((paths[parent[t]] if parent[t] >= 0 else []) + [t])
        bits = np.array([sum(1 << i for i in p) for p in paths])
        depth = np.array([len(p) - 1 for p in paths])
        count = int(rng.integers(0, T + 1))
        see = O.visible(n, count, T, n + T + 5, "mask", bits, window, sinks, n + depth)
        for t in range(T):
            if t >= count:
                assert not see[t].any()
                continue
            # the branch alone: its slots follow the context, its last row sees causally
            m = len(paths[t])
            alone = O.visible(n, m, m, n + m, "causal", None, window, sinks)[-1]
            want = np.zeros(n + T + 5, bool)
            want[:n] = alone[:n]
            want[[n + i for i in paths[t]]] = alone[n:]
            assert np.array_equal(see[t], want), (t, n, window, sinks)
        line = np.arange(T)
        a = O.visible(n, count, T, n + T, "mask", bits, window, sinks, n + line)
        assert np.array_equal(a, O.visible(n, count, T, n + T, "mask", bits, window, sinks))


def test_options_struct_matches_header(pkg):
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dels.h")).read()
    body = re.search(r"typedef struct dels_kv8_options \{(.*?)\} dels_kv8_options;", text, flags=re.S).group(1)
    names = [d.split()[-1].lstrip("*") for d in body.split(";") if d.strip()]
    assert names == [n for n, _ in pkg._lib.Kv8OptionsParams._fields_]


def test_refusals_before_the_gpu(pkg):
    lib = pkg._lib.load()

    def attention(options, block=3, mask=0x9000, window=8, T=4):
        ref = None if options is None else ctypes.byref(pkg._lib.Kv8OptionsParams(*options))
        return lib.dels_kv8_attention_ex(cache(pkg), 0x1000, 4096, 1024, 128, 1, 8, T, 0x3000, None, block, mask, T,
                                         1.0, window, 0, ref, 0x4000, 4096, 1024, 128, 0x5000, 0x6000, 16, None)

    enough = -4                                            # all checks passed but the workspace's
    assert attention(None) == attention((None, 0)) == attention((0x7000, 4)) == attention((0x7000, 0)) == enough
    assert attention((None, 0), block=0, window=0) == enough
    for kw in (dict(block=0), dict(block=1), dict(window=0), dict(block=2, window=0)):
        assert attention((0x7000, 4), **kw) == -1 and b"positions are for a window" in lib.dels_last_error()
    for ld in (3, -1, 1 << 40):
        assert attention((0x7000, ld)) == -1 and b"positions row stride" in lib.dels_last_error()
    assert attention((0x7000, 99), T=65) == -2
    assert attention((0x7000, 4), T=0) == 0


def test_positions_arguments(on_cpu, monkeypatch):  # noqa: F811
    pkg, got = on_cpu
    lib = pkg.kv8._lib.load()
    lib.dels_kv8_attention_ex = lambda *a: got.append(a) or 0
    c, n = small(pkg), torch.zeros(2, dtype=torch.int32)
    q, tree = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int64)
    at, ws = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(1 << 18, dtype=torch.uint8)
    for kw, what in ((dict(positions=at), "for a window over a block mask"),
                     (dict(positions=at, window=4), "for a window over a block mask"),
                     (dict(positions=at, block=tree), "for a window over a block mask"),
                     (dict(positions=at.long(), block=tree, window=4), "positions must be int32"),
                     (dict(positions=at[:, :2], block=tree, window=4), "positions must be int32"),
                     (dict(positions=torch.zeros(3, 2, dtype=torch.int32).t(), block=tree, window=4),
                      "unit column stride")):
        with pytest.raises(ValueError, match=what):
            pkg.kv8_attention(q, c, n, workspace=ws, **kw)
    assert not got
    for given, stride in ((at, 3), (at[:1].expand(2, 3), 0), (torch.zeros(2, 7, dtype=torch.int32)[:, 2:5], 7)):
        pkg.kv8_attention(q, c, n, workspace=ws, block=tree, window=4, sinks=2, positions=given)
        options = got[-1][16]._obj
        assert options.positions == given.data_ptr() and options.ld_positions == stride and got[-1][14:16] == (4, 2)
        assert got[-1][-3:-1] == (ws.data_ptr(), ws.numel())
