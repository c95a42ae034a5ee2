"""CPU tests of the 8-bit cache's argument checks: no kernel is launched, device addresses are fake."""

import ctypes
import types

import pytest
import torch


def cache(pkg, **over):
    f = dict(data=0x10000, num_pages=4, kv_heads=2, head_dim=128, table=0x20000, ld_table=4, batch=2, max_pages=4)
    f.update(over)
    return ctypes.byref(pkg._lib.Kv4CacheParams(*(f[n] for n, _ in pkg._lib.Kv4CacheParams._fields_)))


def rotary(pkg, **over):
    f = dict(cos=0x30000, sin=0x40000, ld=64, positions=100, channels=128, interleaved=0)
    f.update(over)
    return ctypes.byref(pkg._lib.RotaryParams(*(f[n] for n, _ in pkg._lib.RotaryParams._fields_)))


def test_page_and_workspace_sizes(pkg):
    lib = pkg._lib.load()
    assert lib.dels_kv8_page_bytes(128) == 16512 and lib.dels_kv8_page_bytes(64) == 8320
    assert lib.dels_kv8_page_bytes(96) == 0
    base = lib.dels_argmax_rows_ws_bytes(1, 1)
    small, large = (lib.dels_kv8_attention_ws_bytes(b, 16, 32, 8, 128, 512) for b in (1, 64))
    assert base <= small <= large
    assert lib.dels_kv8_attention_ws_bytes(8, 16, 31, 8, 128, 64) == 0
    assert lib.dels_kv8_attention_ws_bytes(8, 16, 32, 8, 96, 64) == 0


def test_rotary_struct_matches_header(pkg):
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dels.h")).read()
    body = re.search(r"typedef struct dels_rotary \{(.*?)\} dels_rotary;", text, flags=re.S).group(1)
    names = [d.split()[-1].lstrip("*") for d in body.split(";") if d.strip()]
    assert names == [n for n, _ in pkg._lib.RotaryParams._fields_]


def test_refusals_before_the_gpu(pkg):
    lib = pkg._lib.load()
    err = lib.dels_last_error

    def append(c, dtype=1, k=0x1000, v=0x2000, stride=128, lengths=0x3000, T=4, r=None, pos=None, ld_pos=4, q=None,
               heads=8, q_out=0x5000, out_stride=128):
        return lib.dels_kv8_append(c, k, 4 * stride, stride, 128, v, 4 * stride, stride, 128, dtype, lengths, None, T,
                                   r, pos, ld_pos, q, 4096, 1024, 128, heads, q_out, 4096, 1024, out_stride, None)

    def attention(c, q=0x1000, dtype=1, heads=8, T=4, lengths=0x3000, block=0, mask=None, ld_mask=0, scale=1.0,
                  window=0, sinks=0, out=0x4000, lse=0x5000, ws=0x6000, ws_bytes=1 << 40):
        return lib.dels_kv8_attention(c, q, 4096, 1024, 128, dtype, heads, T, lengths, None, block, mask, ld_mask,
                                      scale, window, sinks, out, 4096, 1024, 128, lse, ws, ws_bytes, None)

    assert append(None) == -1 and b"cache is NULL" in err()
    assert append(cache(pkg, head_dim=96)) == -2 and b"64 or 128" in err()
    assert append(cache(pkg, kv_heads=0)) == -1 and append(cache(pkg, num_pages=2**31)) == -1
    assert append(cache(pkg, ld_table=3)) == -1 and append(cache(pkg, table=None)) == -1
    assert append(cache(pkg, data=0x10040)) == -3
    assert append(cache(pkg), dtype=9) == -1
    assert append(cache(pkg), k=0x1008) == -3 and b"16-byte" in err()
    assert append(cache(pkg), stride=130) == -3 and append(cache(pkg), stride=-128) == -1
    assert append(cache(pkg), k=None) == -1 and append(cache(pkg), v=None) == -1
    assert append(cache(pkg), lengths=None) == -1
    assert append(cache(pkg), T=-1) == -1 and append(cache(pkg, batch=2**20, kv_heads=2**10), T=2**23) == -2
    assert append(cache(pkg, batch=0)) == 0 and append(cache(pkg), T=0) == 0
    assert append(cache(pkg), r=rotary(pkg, channels=24)) == -1 and b"rotated channels" in err()
    assert append(cache(pkg), r=rotary(pkg, channels=144, ld=72)) == -1
    assert append(cache(pkg), r=rotary(pkg, channels=0)) == -1
    assert append(cache(pkg), r=rotary(pkg, ld=60)) == -1 and append(cache(pkg), r=rotary(pkg, ld=66)) == -3
    assert append(cache(pkg), r=rotary(pkg, cos=0x30004)) == -3 and append(cache(pkg), r=rotary(pkg, sin=None)) == -1
    assert append(cache(pkg), r=rotary(pkg, positions=0)) == -1 and b"no positions" in err()
    assert append(cache(pkg), pos=0x7000) == -1 and b"without a rotary table" in err()
    assert append(cache(pkg), r=rotary(pkg), pos=0x7000, ld_pos=3) == -1
    assert append(cache(pkg), q=0x8000) == -1 and b"without a rotary table" in err()
    assert append(cache(pkg), r=rotary(pkg), q=0x8000, heads=7) == -1 and b"query heads" in err()
    assert append(cache(pkg), r=rotary(pkg), q=0x8000, q_out=None) == -1
    assert append(cache(pkg), r=rotary(pkg), q=0x8000, out_stride=132) == -3
    assert append(cache(pkg), r=rotary(pkg), q=0x8008) == -3
    assert lib.dels_kv8_read(cache(pkg), None, None, 4, 0x1000, 0x2000, 1, None) == -1
    assert lib.dels_kv8_read(cache(pkg), 0x3000, None, 4, 0x1004, 0x2000, 1, None) == -3

    assert attention(cache(pkg), dtype=0) == -1
    assert attention(cache(pkg), heads=7) == -1 and b"query heads" in err()
    assert attention(cache(pkg), block=4) == -1 and attention(cache(pkg), block=-1) == -1
    assert attention(cache(pkg), block=3) == -1 and b"mask is NULL" in err()
    assert attention(cache(pkg), block=3, mask=0x9000, ld_mask=3) == -1
    assert attention(cache(pkg), block=3, mask=0x9000, ld_mask=99, T=65) == -2
    assert attention(cache(pkg), scale=float("inf")) == -1 and b"finite" in err()
    assert attention(cache(pkg), window=-1) == -1 and attention(cache(pkg), window=4, sinks=-1) == -1
    assert attention(cache(pkg), sinks=4) == -1 and b"window" in err()
    assert attention(cache(pkg), lengths=None) == -1 and attention(cache(pkg), lse=None) == -1
    assert attention(cache(pkg), out=0x4004) == -3
    assert attention(cache(pkg), ws_bytes=16) == -4 and attention(cache(pkg), ws=None) == -4
    assert attention(cache(pkg), T=2**23, heads=2**10) == -2
    assert attention(cache(pkg), T=0) == 0


def test_workspace_of_the_longest_block_serves_shorter_ones(pkg):
    lib = pkg._lib.load()
    for batch, q_heads, heads in ((1, 8, 8), (3, 32, 8), (40, 32, 8), (7, 64, 8)):
        for max_pages in (1, 40, 2000):
            sizes = [lib.dels_kv8_attention_ws_bytes(batch, T, q_heads, heads, 128, max_pages) for T in range(1, 700)]
            assert all(x <= y for x, y in zip(sizes, sizes[1:]))


@pytest.fixture
def on_cpu(pkg, monkeypatch):
    """The wrappers' checks with CPU tensors in the GPU's place, and a library whose calls succeed."""
    monkeypatch.setattr(pkg.kv4, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(pkg.kv8, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(pkg.kv8, "_stream_ptr", lambda device: 0)
    monkeypatch.setattr(pkg.ops, "_stream_ptr", lambda device: 0)
    got = []
    lib = types.SimpleNamespace(dels_kv8_append=lambda *a: got.append(a) or 0, dels_kv8_read=lambda *a: 0,
                                dels_kv8_attention_ws_bytes=lambda *a: 1 << 18,
                                dels_kv8_attention=lambda *a: got.append(a) or 0)
    monkeypatch.setattr(pkg.kv8._lib, "load", lambda: lib)
    return pkg, got


def small(pkg, batch=2):
    return pkg.KV8Cache(torch.zeros(4, 2, 8320, dtype=torch.uint8), torch.zeros(batch, 2, dtype=torch.int32), 64)


def test_a_cache_of_the_other_format_is_refused(on_cpu):
    pkg, _ = on_cpu
    c8 = small(pkg)
    c4 = pkg.KV4Cache(torch.zeros(4, 2, 4352, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), 64)
    kv, n = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    lse, w = torch.zeros(2, 3, 2), torch.zeros(2, 2, 128)
    for call in (lambda: pkg.kv8_append(c4, kv, kv, n), lambda: pkg.kv8_read(c4, n, 3),
                 lambda: pkg.kv8_attention(kv, c4, n), lambda: pkg.kv4_append(c8, kv, kv, n),
                 lambda: pkg.kv4_read(c8, n, 3), lambda: pkg.kv4_attention(kv, c8, n),
                 lambda: pkg.kv4_weights(kv, c8, n, lse, w), lambda: pkg.kv4_evict(c8, n, w, 10)):
        with pytest.raises(TypeError, match="bits a value"):
            call()
    with pytest.raises(ValueError, match="data must be uint8"):
        pkg.KV8Cache(c4.data, c4.block_table, 64)


def test_rotary_tables_that_are_refused(on_cpu):
    pkg, _ = on_cpu
    t = torch.zeros(10, 32)
    for cos, sin, what in ((t.double(), t, "float32"), (t, t[0], "positions, channels"), (t, t[:9], "one shape"),
                           (t[:, :20], t[:, :20], "multiple of 16"), (t[:, :4], t[:, :4], "multiple of 16"),
                           (t.t().contiguous().t(), t, "unit column stride"),
                           (t, torch.zeros(10, 64)[:, :32], "one row stride"),
                           (torch.zeros(70).as_strided((3, 32), (16, 1)), torch.zeros(3, 32), "overlapping rows")):
        with pytest.raises(ValueError, match=what):
            pkg.RotaryTable(cos, sin)
    assert pkg.RotaryTable(t, t).channels == 64


def test_append_arguments(on_cpu):
    pkg, got = on_cpu
    cache, n = small(pkg), torch.zeros(2, dtype=torch.int32)
    kv, q = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    r = pkg.RotaryTable(torch.zeros(10, 32), torch.zeros(10, 32))
    at = torch.zeros(2, 3, dtype=torch.int32)
    for kw, error, what in ((dict(q=q), ValueError, "for a rotary table"),
                            (dict(positions=at), ValueError, "for a rotary table"),
                            (dict(rotary=r, q_out=q), ValueError, "q_out is for q"),
                            (dict(rotary=r, q=q.float()), TypeError, "q dtype"),
                            (dict(rotary=r, q=q[:, :2]), ValueError, "q must be"),
                            (dict(rotary=r, q=q[:, :, :3]), ValueError, "q must be"),
                            (dict(rotary=r, q=q[:, :, :0]), ValueError, "q must be"),
                            (dict(rotary=r, q=q, q_out=q[:, :, :2]), ValueError, "q_out must be"),
                            (dict(rotary=r, positions=at.long()), ValueError, "positions must be int32"),
                            (dict(rotary=r, positions=at[:, :2]), ValueError, "positions must be int32"),
                            (dict(rotary=r, positions=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError,
                             "unit column stride"),
                            (dict(rotary=pkg.RotaryTable(torch.zeros(10, 40), torch.zeros(10, 40))), ValueError,
                             "80 rotated channels")):
        with pytest.raises(error, match=what):
            pkg.kv8_append(cache, kv, kv, n, **kw)
    with pytest.raises(ValueError, match="one shape and dtype"):
        pkg.kv8_append(cache, kv, kv.float(), n)
    assert not got
    assert pkg.kv8_append(cache, kv, kv, n) is None
    out = pkg.kv8_append(cache, kv, kv, n, rotary=r, q=q)
    assert out.shape == q.shape and out.data_ptr() != q.data_ptr()
    assert pkg.kv8_append(cache, kv, kv, n, rotary=r, q=q, q_out=q) is q
    # one row of positions for all sequences is a stride of zero
    pkg.kv8_append(cache, kv, kv, n, rotary=r, positions=at[:1].expand(2, 3))
    assert got[-1][15] == 0
    pkg.kv8_append(cache, kv, kv, n, rotary=r, positions=torch.zeros(2, 7, dtype=torch.int32)[:, 2:5])
    assert got[-1][15] == 7


def test_attention_arguments(on_cpu, monkeypatch):
    pkg, got = on_cpu
    cache, n = small(pkg), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    for kw, what in ((dict(window=0), "window must be"), (dict(window=5, sinks=-1), "sinks at least"),
                     (dict(sinks=3), "sinks are for a window"), (dict(block="window"), "block must be one of"),
                     (dict(out=q[:, :1]), "out must be"), (dict(lse=torch.zeros(2, 3)), "lse must be")):
        with pytest.raises(ValueError, match=what):
            pkg.kv8_attention(q, cache, n, workspace=torch.zeros(1, dtype=torch.uint8), **kw)
    taken = []

    def shared(device, need, stream):
        taken.append(need)
        return torch.zeros(need, dtype=torch.uint8)

    monkeypatch.setattr(pkg.kv8._WORKSPACES, "get", shared)
    for capturing in (False, True):                        # a captured call has a workspace of its own
        monkeypatch.setattr(pkg.kv8, "_capturing", lambda: capturing)
        pkg.kv8_attention(q, cache, n, window=7, sinks=2)
        assert len(taken) == 1 and got[-1][14:16] == (7, 2) and got[-1][-2] >= 1 << 18
    mine = torch.zeros(1 << 18, dtype=torch.uint8)
    pkg.kv8_attention(q, cache, n, workspace=mine)
    assert got[-1][-3:-1] == (mine.data_ptr(), mine.numel()) and got[-1][14:16] == (0, 0)
    with pytest.raises(ValueError, match="workspace must be"):
        pkg.kv8_attention(q, cache, n, workspace=torch.zeros(1 << 18))
    # numbers past 64 bits arrive as numbers past every slot
    for big in (2**62, 2**63, 2**64 + 5):
        pkg.kv8_attention(q, cache, n, window=big, sinks=big, workspace=mine)
        assert min(got[-1][14:16]) > 1 << 31 and max(got[-1][14:16]) < 1 << 63
