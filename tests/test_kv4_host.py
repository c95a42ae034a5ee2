"""CPU tests of the 4-bit cache's C ABI checks: no kernel is launched, device addresses are fake."""

import ctypes


def cache(pkg, **over):
    f = dict(data=0x10000, num_pages=4, kv_heads=2, head_dim=128, table=0x20000, ld_table=4, batch=2, max_pages=4)
    f.update(over)
    return ctypes.byref(pkg._lib.Kv4CacheParams(*(f[n] for n, _ in pkg._lib.Kv4CacheParams._fields_)))


def test_page_and_workspace_sizes(pkg):
    lib = pkg._lib.load()
    assert lib.dels_kv4_page_bytes(128) == 8576 and lib.dels_kv4_page_bytes(64) == 4352
    assert lib.dels_kv4_page_bytes(96) == 0
    base = lib.dels_argmax_rows_ws_bytes(1, 1)
    assert lib.dels_kv4_attention_ws_bytes(8, 16, 32, 8, 128, 64) >= base
    small, large = (lib.dels_kv4_attention_ws_bytes(b, 16, 32, 8, 128, 512) for b in (1, 64))
    assert base <= small <= large
    assert lib.dels_kv4_evict_ws_bytes(2, 8, 100) >= base + 2 * 8 * 100 * 4
    assert lib.dels_kv4_evict_ws_bytes(2**23, 2**23, 2**30) == 0


def test_cache_struct_matches_header(pkg):
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dels.h")).read()
    body = re.search(r"typedef struct dels_kv4_cache \{(.*?)\} dels_kv4_cache;", text, flags=re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [d.split()[-1].lstrip("*") for d in body.split(";") if d.strip()]
    assert names == [n for n, _ in pkg._lib.Kv4CacheParams._fields_]


def test_refusals_before_the_gpu(pkg):
    lib = pkg._lib.load()
    err = lib.dels_last_error

    def append(c, dtype=1, k=0x1000, stride=128, lengths=0x3000, T=4):
        return lib.dels_kv4_append(c, k, 4 * stride, stride, 128, 0x2000, 4 * stride, stride, 128, dtype, lengths,
                                   None, T, None)

    def attention(c, q=0x1000, dtype=1, heads=8, T=4, lengths=0x3000, block=0, mask=None, ld_mask=0, scale=1.0,
                  out=0x4000, lse=0x5000, ws=0x6000, ws_bytes=1 << 40):
        return lib.dels_kv4_attention(c, q, 4096, 1024, 128, dtype, heads, T, lengths, None, block, mask, ld_mask,
                                      scale, out, 4096, 1024, 128, lse, ws, ws_bytes, None)

    def evict(c, keep=4, recent=0, lengths=0x3000, out_lengths=0x4000, w=0x5000, ow=0x7000, ws_bytes=1 << 40):
        return lib.dels_kv4_evict(c, lengths, w, keep, recent, out_lengths, ow, 0x8000, 0x6000, ws_bytes, None)

    assert append(None) == -1 and b"cache is NULL" in err()
    assert append(cache(pkg, head_dim=96)) == -2 and b"64 or 128" in err()
    assert append(cache(pkg, kv_heads=0)) == -1
    assert append(cache(pkg, num_pages=2**31)) == -1
    assert append(cache(pkg, ld_table=3)) == -1 and b"table row stride" in err()
    assert append(cache(pkg, table=None)) == -1
    assert append(cache(pkg, data=0x10040)) == -3
    assert append(cache(pkg), dtype=9) == -1
    assert append(cache(pkg), k=0x1008) == -3 and b"16-byte" in err()
    assert append(cache(pkg), stride=130) == -3
    assert append(cache(pkg), stride=-128) == -1
    assert append(cache(pkg), k=None) == -1 and append(cache(pkg), lengths=None) == -1
    assert append(cache(pkg), T=-1) == -1 and append(cache(pkg, batch=2**20, kv_heads=2**10), T=2**23) == -2
    assert append(cache(pkg, batch=0)) == 0 and append(cache(pkg), T=0) == 0
    assert lib.dels_kv4_read(cache(pkg), None, None, 4, 0x1000, 0x2000, 1, None) == -1
    assert lib.dels_kv4_read(cache(pkg), 0x3000, None, 4, 0x1004, 0x2000, 1, None) == -3

    assert attention(cache(pkg), dtype=0) == -1
    assert attention(cache(pkg), heads=7) == -1 and b"query heads" in err()
    assert attention(cache(pkg), block=4) == -1 and attention(cache(pkg), block=-1) == -1
    assert attention(cache(pkg), block=3) == -1 and b"mask is NULL" in err()
    assert attention(cache(pkg), block=3, mask=0x9000, ld_mask=3) == -1
    assert attention(cache(pkg), block=3, mask=0x9000, ld_mask=99, T=65) == -2
    assert attention(cache(pkg), scale=float("inf")) == -1 and b"finite" in err()
    assert attention(cache(pkg), lengths=None) == -1 and attention(cache(pkg), lse=None) == -1
    assert attention(cache(pkg), out=0x4004) == -3
    assert attention(cache(pkg), ws_bytes=16) == -4 and attention(cache(pkg), ws=None) == -4
    assert attention(cache(pkg), T=2**23, heads=2**10) == -2
    assert attention(cache(pkg), T=0) == 0
    assert lib.dels_kv4_weights(cache(pkg), 0x1000, 4096, 1024, 128, 1, 8, 4, 0x3000, None, None, 0, None, 0, 1.0,
                                None, 0x5000, 0x5000, None) == -1

    assert evict(cache(pkg), keep=0) == -1 and evict(cache(pkg), recent=-1) == -1
    assert evict(cache(pkg), out_lengths=0x3000) == -1 and b"one of the inputs" in err()
    assert evict(cache(pkg), ow=0x5000) == -1
    assert evict(cache(pkg), ws_bytes=4) == -4
    assert evict(cache(pkg), w=None) == -1


def test_workspace_of_the_longest_block_serves_shorter_ones(pkg):
    lib = pkg._lib.load()
    for batch, q_heads, heads in ((1, 8, 8), (3, 32, 8), (40, 32, 8), (7, 64, 8)):
        for max_pages in (1, 40, 2000):
            sizes = [lib.dels_kv4_attention_ws_bytes(batch, T, q_heads, heads, 128, max_pages) for T in range(1, 700)]
            assert all(x <= y for x, y in zip(sizes, sizes[1:]))
