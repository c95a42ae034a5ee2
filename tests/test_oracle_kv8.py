"""CPU tests of the 8-bit cache's oracle: its rounding, layout, rotation and visibility by closed forms."""

import numpy as np
import pytest
import torch

from oracle import kv8 as O


def test_codes_are_torchs_e4m3():
    x = np.concatenate([np.linspace(-448, 448, 20011), O.LEVELS, O.MIDDLES, -O.MIDDLES,
                        np.nextafter(O.MIDDLES, 0), np.nextafter(O.MIDDLES, 500), np.geomspace(1e-6, 448, 5000)])
    x = x.astype(np.float32)
    want = torch.tensor(x).to(torch.float8_e4m3fn)
    assert np.array_equal(O.encode(x.astype(np.float64)), want.view(torch.uint8).numpy())
    codes = np.arange(256, dtype=np.uint8)
    got, ref = O.decode(codes), torch.tensor(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(got, ref, equal_nan=True)


@pytest.mark.parametrize("top,e", [(0.0, 63), (448.0, 127), (448.1, 128), (224.0, 126), (224.01, 127), (1e-30, 63),
                                   (448 * 2.0 ** 64, 191), (1e30, 191), (1.0, 119)])
def test_exponents(top, e):
    assert O.exponent(top) == e


def test_a_page_holds_every_slot_once():
    for D in (64, 128):
        assert sorted(O.place(s) for s in range(32)) == list(range(32))
        data = np.arange(O.page_bytes(D) * 3, dtype=np.uint64).reshape(3, 1, -1)
        # each byte of keys and values is read by exactly one (slot, channel)
        marks = (data % 251).astype(np.uint8)
        kc, ke, vc, ve, bad = O.unpack(marks, np.array([[2]]), D)
        seen = np.zeros(128 * D, int)
        for c in range(D):
            for j in range(64):
                u, s = j // 32, j % 32
                kat = 32 * D * u + 512 * (c // 16) + 16 * O.place(s) + c % 16
                vat = 64 * D + 32 * D * u + 16 * D * (s // 16) + 16 * c + s % 16
                seen[kat] += 1
                seen[vat] += 1
                assert kc[0, 0, j, c] == marks[2, 0, kat] and vc[0, 0, j, c] == marks[2, 0, vat]
        assert (seen == 1).all()


def test_rotation_is_a_complex_product():
    g = np.random.default_rng(1)
    x = g.standard_normal((5, 2, 32)).astype(np.float32)
    angle = g.standard_normal((9, 8))
    at = np.array([[0, 8], [3, 3], [1, 2], [-1, 4], [9, 0]])
    for interleaved in (False, True):
        y = O.rotate(x, np.cos(angle), np.sin(angle), at, interleaved)
        pick = (slice(0, 16, 2), slice(1, 16, 2)) if interleaved else (slice(0, 8), slice(8, 16))
        z = (x[..., pick[0]] + 1j * x[..., pick[1]]) * np.exp(1j * angle[np.clip(at, 0, 8)])
        ok = (at >= 0) & (at < 9)
        assert np.allclose(y[ok][:, pick[0]], z.real[ok], atol=1e-6)
        assert np.allclose(y[ok][:, pick[1]], z.imag[ok], atol=1e-6)
        assert np.isnan(y[~ok][:, :16]).all() and np.array_equal(y[..., 16:], x[..., 16:])


def test_append_keeps_the_larger_exponent():
    """Kept rows move to a larger exponent of new ones; a smaller one of new rows gives way."""
    D = 64
    state = [np.zeros((1, 64, D), np.uint8), np.zeros((1, 2), np.uint8), np.zeros((1, 64, D), np.uint8),
             np.zeros((1, 2), np.uint8), np.zeros((1, 64), bool)]
    one = np.ones((1, 1, D))
    O.append(state, one, 4 * one, 0, 1)
    assert state[1][0, 0] == 119 and state[3][0, 0] == 121
    O.append(state, 300 * one, one, 1, 1)
    assert state[1][0, 0] == 127 and state[3][0, 0] == 121
    x = O.values(state[0][None], state[1][None], state[4][None])[0, 0]
    assert np.all(x[0] == 1.0) and np.all(x[1] == 288.0 + 0.0 * x[1])
    # the next block starts anew; a row that is not finite takes part in neither exponent
    O.append(state, one, np.nan * one, 32, 1)
    assert state[1][0, 1] == 63 and state[4][0, 32] and state[3][0, 1] == 63
    # a first row again: what was there is forgotten
    O.append(state, 0.5 * one, one, 0, 1)
    assert state[1][0, 0] == 118 and not state[4][0, :32].any()


def test_visibility():
    see = O.visible(5, 3, 4, 10, "causal", window=4, sinks=1)
    assert see[0].nonzero()[0].tolist() == [0, 2, 3, 4, 5]
    assert see[2].nonzero()[0].tolist() == [0, 4, 5, 6, 7]
    assert not see[3].any()
    assert O.visible(5, 3, 3, 10, "none", window=2)[1].nonzero()[0].tolist() == []
    assert O.visible(5, 3, 3, 10, "none", window=3)[1].nonzero()[0].tolist() == [4]
    tree = O.visible(2, 3, 3, 8, "mask", np.array([1, 3, 5]))
    assert [r.nonzero()[0].tolist() for r in tree] == [[0, 1, 2], [0, 1, 2, 3], [0, 1, 2, 4]]


def test_attention_against_torch():
    g = np.random.default_rng(2)
    q, K, V = g.standard_normal((1, 4, 4, 16)), g.standard_normal((1, 2, 64, 16)), g.standard_normal((1, 2, 64, 16))
    out, lse, _, _ = O.attention(q, K, V, [40], [4], "causal", 0.3, window=20, sinks=3)
    see = torch.tensor(O.visible(40, 4, 4, 64, "causal", window=20, sinks=3))
    for hq in range(4):
        x = torch.tensor(q[0, :, hq] @ K[0, hq // 2].T * 0.3).masked_fill(~see, float("-inf"))
        assert np.allclose(out[0, :, hq], (x.softmax(-1).numpy() @ V[0, hq // 2]))
        assert np.allclose(lse[0, :, hq], torch.logsumexp(x, -1).numpy())
