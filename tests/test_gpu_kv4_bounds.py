"""GPU tests of the 4-bit cache's attention at the bound that two bf16 parts of each weight allow.

The bound goes by the output's type (oracle/kv4.py, ``output_range``): one part alone is
outside of it, as the CPU tests of the bound show, most clearly where scores are small and
their own error leaves room for nothing else.
"""

import numpy as np
import pytest
import torch

from oracle import kv4 as O
from test_gpu_kv4 import ATTENTION, attention_inputs, contents, ints, say, score_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,sharp", [("bf16", 1.0), ("f16", 1.0), ("bf16", 2.0 ** -6), ("f16", 2.0 ** -6)])
@pytest.mark.parametrize("B,T,HQ,H,D,pages,_,block,lengths,counts", ATTENTION)
def test_outputs_are_within_the_two_parts_bound(pkg, dev, B, T, HQ, H, D, pages, _, block, lengths, counts, dtype,
                                                 sharp):
    say("bound", B, T, HQ, H, D, pages, dtype, block, lengths, counts, sharp)
    cache, q, masks = attention_inputs(pkg, dev, B, T, HQ, H, D, pages, dtype, block, lengths, counts,
                                        seed=3 + B * T, sharp=sharp)
    out, lse = pkg.kv4_attention(q.to(dev), cache, ints(lengths, dev),
                                 block=block if masks is None else masks.to(dev), counts=ints(counts, dev))
    torch.cuda.synchronize()
    K, V = contents(cache)
    q64, count = q.double().numpy(), [T] * B if counts is None else counts
    ro, rl, weight, mass = O.attention(q64, K, V, lengths, count, block, D ** -0.5,
                                       None if masks is None else masks.numpy())
    lo, hi = O.output_range(ro, weight, score_error(q64, mass, dtype, D ** -0.5), dtype)
    got = out.double().cpu().numpy()
    assert np.all((lo <= got) & (got <= hi))
