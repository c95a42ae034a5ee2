"""CPU tests of what the 4-bit cache's Python calls hand to the C ABI: no kernel is launched."""

import types

import pytest
import torch

import test_kv4_host as host


@pytest.fixture
def on_cpu(pkg, monkeypatch):
    """The wrappers' checks with CPU tensors in the GPU's place."""
    monkeypatch.setattr(pkg.kv4, "_require_cuda", lambda *a: None)
    return pkg


def last_row_ends(stride, rows, columns):
    return (rows - 1) * stride + columns


@pytest.mark.parametrize("T", [1, 5, 64])
def test_a_block_mask_is_read_inside_its_storage(pkg, T):
    cache = types.SimpleNamespace(_index=-1, batch=4, device="cpu")
    for mask in (torch.zeros(1, T, dtype=torch.int64).expand(4, T), torch.zeros(4, T, dtype=torch.int64),
                 torch.zeros(4, T + 3, dtype=torch.int64)[:, :T]):
        mode, p, ld = pkg.kv4._block_args(mask, cache, T)
        assert mode == 3 and p == mask.data_ptr()
        assert last_row_ends(ld, 4, T) <= mask.untyped_storage().nbytes() // 8
        assert ld == mask.stride(0)
    if T > 1:
        with pytest.raises(ValueError, match="overlapping rows"):
            pkg.kv4._block_args(torch.zeros(T + 3, dtype=torch.int64).as_strided((4, T), (1, 1)), cache, T)


def test_a_page_table_is_read_inside_its_storage(on_cpu):
    data = torch.zeros(5, 2, 4352, dtype=torch.uint8)
    for table in (torch.zeros(1, 3, dtype=torch.int32).expand(4, 3), torch.zeros(4, 3, dtype=torch.int32),
                  torch.zeros(4, 7, dtype=torch.int32)[:, 2:5], torch.zeros(4, 1, dtype=torch.int32),
                  torch.zeros(1, 1, dtype=torch.int32).expand(4, 1), torch.zeros(1, 3, dtype=torch.int32)):
        params = on_cpu.KV4Cache(data, table, 64)._params
        room = table.untyped_storage().nbytes() // 4 - table.storage_offset()
        assert last_row_ends(params.ld_table, table.shape[0], table.shape[1]) <= room
    with pytest.raises(ValueError, match="overlapping rows"):
        on_cpu.KV4Cache(data, torch.zeros(9, dtype=torch.int32).as_strided((4, 3), (2, 1)), 64)


def test_one_row_for_all_sequences_is_a_stride_of_zero(pkg):
    lib = pkg._lib.load()
    assert lib.dels_kv4_append(host.cache(pkg, ld_table=0), 0x1000, 512, 128, 128, 0x2000, 512, 128, 128, 1, 0x3000,
                               None, 0, None) == 0
    # past the stride checks: the workspace is refused next
    for ld in (0, 4):
        assert lib.dels_kv4_attention(host.cache(pkg), 0x1000, 4096, 1024, 128, 1, 8, 4, 0x3000, None, 3, 0x9000, ld,
                                      1.0, 0x4000, 4096, 1024, 128, 0x5000, None, 0, None) == -4


class Answers:
    """A library whose calls succeed; what they got for a workspace is written down."""

    def __init__(self):
        self.got = []

    def dels_kv4_attention_ws_bytes(self, *a):
        return 1 << 18

    dels_kv4_evict_ws_bytes = dels_kv4_attention_ws_bytes

    def dels_kv4_attention(self, *a):
        self.got.append(a[-3:-1])
        return 0

    dels_kv4_evict = dels_kv4_attention


def test_captured_calls_do_not_use_the_streams_shared_workspace(on_cpu, monkeypatch):
    lib, taken = Answers(), []
    kv4, cpu = on_cpu.kv4, torch.device("cpu")
    monkeypatch.setattr(kv4._lib, "load", lambda: lib)
    monkeypatch.setattr(kv4, "_stream_ptr", lambda device: 0)
    monkeypatch.setattr(on_cpu.ops, "_stream_ptr", lambda device: 0)

    def shared(device, need, stream):
        taken.append(need)
        return torch.zeros(need, dtype=torch.uint8)

    monkeypatch.setattr(kv4._WORKSPACES, "get", shared)
    cache = on_cpu.KV4Cache(torch.zeros(4, 2, 4352, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), 64)
    q, n = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device=cpu), torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(2, 2, 128)
    for capturing in (False, True):
        monkeypatch.setattr(kv4, "_capturing", lambda: capturing)
        on_cpu.kv4_attention(q, cache, n)
        on_cpu.kv4_evict(cache, n, w, 10)
        assert len(taken) == 2                       # of the calls that no graph captured
        assert all(p and size >= 1 << 18 for p, size in lib.got)
    mine = torch.zeros(1 << 18, dtype=torch.uint8)
    on_cpu.kv4_attention(q, cache, n, workspace=mine)
    on_cpu.kv4_evict(cache, n, w, 10, workspace=mine)
    assert lib.got[-2:] == [(mine.data_ptr(), mine.numel())] * 2 and len(taken) == 2
    with pytest.raises(ValueError, match="workspace must be"):
        on_cpu.kv4_attention(q, cache, n, workspace=torch.zeros(1 << 18))


def test_keys_and_values_that_are_read_are_tensors_of_their_own(on_cpu, monkeypatch):
    """Either outlives the other alone, and takes in-place operations that autograd records."""
    kv4 = on_cpu.kv4
    lib = types.SimpleNamespace(dels_kv4_read=lambda *a: 0)
    monkeypatch.setattr(kv4._lib, "load", lambda: lib)
    monkeypatch.setattr(kv4, "_stream_ptr", lambda device: 0)
    cache = on_cpu.KV4Cache(torch.zeros(4, 2, 4352, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), 64)
    k, v = on_cpu.kv4_read(cache, torch.zeros(2, dtype=torch.int32), 5, dtype=torch.float32)
    for x in (k, v):
        assert x.shape == (2, 5, 2, 64) and x.is_contiguous()
        assert x.untyped_storage().nbytes() == x.numel() * 4
        x.add_(torch.ones(64, requires_grad=True))
    assert k.untyped_storage().data_ptr() != v.untyped_storage().data_ptr()


def test_a_cache_of_no_heads_is_refused(on_cpu):
    with pytest.raises(ValueError, match="one key/value head"):
        on_cpu.KV4Cache(torch.zeros(4, 0, 4352, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), 64)
