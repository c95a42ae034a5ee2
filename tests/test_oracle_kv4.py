"""CPU tests of the 4-bit cache's oracle: closed forms, its format, and torch's own attention."""

import math

import numpy as np
import pytest
import torch

from oracle import kv4 as O


def test_codes_are_nearest_levels_with_ties_to_even():
    assert list(O.decode(np.arange(16, dtype=np.uint8))) == [0, .5, 1, 1.5, 2, 3, 4, 6,
                                                             0, -.5, -1, -1.5, -2, -3, -4, -6]
    ties = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0])
    assert list(O.decode(O.encode(ties))) == [0, 1, 1, 2, 2, 4, 4]
    assert list(O.decode(O.encode(-ties))) == [0, -1, -1, -2, -2, -4, -4]
    y = np.random.default_rng(0).uniform(-7, 7, 4000)
    got = O.decode(O.encode(y))
    best = np.abs(y[:, None] - np.concatenate([O.LEVELS, -O.LEVELS])[None]).min(1)
    assert np.allclose(np.abs(y - got), best)


@pytest.mark.parametrize("amax,exponent", [(7.0, 127), (7.0001, 128), (3.5, 126), (3.6, 127), (1.0, 125), (0.0, 1),
                                           (2.0 ** -140, 1), (1e38, 251), (np.inf, 252), (3.4e38, 252)])
def test_key_exponent_is_the_smallest_whose_sevenfold_holds(amax, exponent):
    x = np.zeros(32)
    x[5] = -amax
    codes, e = O.encode_keys(x)
    assert e[0] == exponent
    if 0 < amax < 1e38 and amax > 1e-30:
        assert abs(O.key_values(codes, e)[5]) >= amax * 6 / 7 - 1e-9


def test_no_element_is_off_by_more_than_its_step_allows():
    rng = np.random.default_rng(1)
    k = rng.normal(size=(50, 128)) * 10.0 ** rng.uniform(-3, 3, size=(50, 1))
    codes, e = O.encode_keys(k)
    err = np.abs(O.key_values(codes, e) - k).reshape(50, 4, 32)
    assert np.all(err <= 2.0 ** (e[..., None].astype(float) - 127))          # half the widest step, 2
    codes, s = O.encode_values(k)
    assert np.all(np.abs(O.value_values(codes, s) - k) <= s[:, None] * (1 + 6 * 2.0 ** -8))


def test_nan_and_infinity():
    x = np.zeros(64)
    x[0], x[1], x[40] = np.nan, -np.inf, 2.0
    codes, e = O.encode_keys(x)
    y = O.key_values(codes, e)
    assert y[0] == 0 and y[1] == -6 * 2.0 ** 125 and y[40] == 2.0
    codes, s = O.encode_values(x)
    assert np.isfinite(O.value_values(codes, s)).all()


def test_attention_is_torch_softmax_attention():
    rng = np.random.default_rng(2)
    B, T, HQ, H, D, S = 2, 3, 6, 2, 8, 20
    q, K, V = rng.normal(size=(B, T, HQ, D)), rng.normal(size=(B, H, S, D)), rng.normal(size=(B, H, S, D))
    lengths, counts = [11, 0], [3, 2]
    out, lse, weight, _ = O.attention(q, K, V, lengths, counts, "causal", 0.3)
    for b in range(B):
        n, c = lengths[b], counts[b]
        mask = torch.ones(c, n + c, dtype=torch.bool).tril(n)
        for hq in range(HQ):
            x = torch.tensor(q[b, :c, hq] @ K[b, hq // 3, :n + c].T * 0.3).masked_fill(~mask, -math.inf)
            assert np.allclose(out[b, :c, hq], torch.softmax(x, -1).numpy() @ V[b, hq // 3, :n + c])
            assert np.allclose(lse[b, :c, hq], torch.logsumexp(x, -1).numpy())
    assert np.all(out[1, 2] == 0) and np.all(lse[1, 2] == -np.inf)
    assert np.all(weight >= np.abs(out) - 1e-12)


def test_weights_of_full_acceptance_sum_to_the_rows():
    rng = np.random.default_rng(3)
    q, K = rng.normal(size=(1, 4, 4, 8)), rng.normal(size=(1, 2, 16, 8))
    _, lse, _, _ = O.attention(q, K, K, [9], [4], "full", 1.0)
    w, added, _ = O.weights(q, K, [9], [4], [4], "full", 1.0, lse, np.full((1, 2, 16), 5.0))
    assert np.allclose(added.sum(-1), 4 * 2) and np.all(w[..., 13:] == 0)
    assert np.allclose(w[..., :9] - added[..., :9], 5.0) and np.allclose(w[..., 9:13], added[..., 9:13])


def test_evict_fills_places_in_order():
    w = np.array([5, 1, 5, 0, 9, 5, 5, 2, 3, 4.0])
    assert list(O.evict(w, 10, 4, 1)) == [0, 4, 2, 9]          # stays: 4, 0, 2 by weight (ties lowest), 9 as recent
    assert list(O.evict(w, 10, 3, 3)) == [7, 8, 9]
    assert list(O.evict(w, 2, 4, 1)) == [0, 1, -1, -1]
    assert list(O.evict(np.full(6, np.nan), 6, 2, 0)) == [0, 1]


def test_page_layout_by_hand():
    """One code and one scale at a time, at the byte that the format names."""
    D = 64
    for j in (0, 3, 4, 9, 31, 32, 63):
        page = np.zeros(O.page_bytes(D), np.uint8)
        page[j * 32 + 5] = 0x70
        page[32 * D + 64 + 16 * (j // 8 % 4) + 4 * (j % 4) + 2 * (j // 32) + (j // 4 % 2)] = 130
        page[34 * D + (j // 8) * 4 * D + 4 * 17 + (j % 8) // 2] = 0xA0 if j % 2 else 0x0A
        page[66 * D + 2 * j + 1] = 0x3F
        kc, ke, vc, vs = O.unpack_page(page, D)
        assert kc[j, 11] == 7 and kc.sum() == 7
        assert ke[j, 1] == 130 and ke.sum() == 130
        assert vc[j, 17] == 10 and vc.sum() == 10
        assert vs[j] == 0.5 and vs.sum() == 0.5
