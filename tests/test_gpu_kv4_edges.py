"""GPU tests of the 4-bit cache's calls at the edges of what they take."""

import pytest
import torch

from test_gpu_kv4 import attention_inputs, ints, say

pytestmark = pytest.mark.gpu


def test_one_tree_and_one_row_of_pages_for_all_sequences(pkg, dev):
    """Expanded masks and tables: as their copies."""
    say("expanded mask and table")
    B, T, HQ, H, D = 5, 7, 4, 2, 64
    cache, q, _ = attention_inputs(pkg, dev, 1, T, HQ, H, D, 3, "bf16", "full", [130], None, 12)
    qd = q.expand(B, T, HQ, D).contiguous().to(dev)
    table = cache.block_table.expand(B, -1)
    mask = torch.tensor([(1 << t) | (t and 1) for t in range(T)], device=dev)[None]
    n = ints([130, 64, 5, 0, 100], dev)
    made = []
    for tab, m in ((table, mask.expand(B, T)), (table.contiguous(), mask.repeat(B, 1))):
        c = pkg.KV4Cache(cache.data, tab, D)
        out, lse = pkg.kv4_attention(qd, c, n, block=m)
        w = pkg.kv4_weights(qd, c, n, lse, torch.zeros(B, H, c.slots, device=dev), block=m)
        made.append((out, lse, w, *pkg.kv4_read(c, n, 9)))
    torch.cuda.synchronize()
    for x, y in zip(*made):                                # as bits: the slots past 136 hold NaN
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    assert torch.isfinite(made[0][1]).all()
