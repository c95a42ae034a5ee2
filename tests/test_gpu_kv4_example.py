"""GPU test of the example loop: drafts verified over 4-bit caches, with and without eviction."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(pkg):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_kv4.py")
    spec = importlib.util.spec_from_file_location("verify_kv4", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_ids_are_the_targets_own(example, dev):
    """Without eviction every id is the target's first choice after the ids before it.

    The ids go through the target once more, as one prompt.  Its matrix products may then
    sum in another order, which moves logits by bf16 roundings, and where a key or value
    falls to another code by a fraction of one slot's share: 1/16 of the largest logit covers both.
    """
    print("case kv4 example, no eviction", flush=True)
    target, prompt, ids, count, held = example.main("--batch 3 --prompt 70 --rounds 9 --draft 5 --keep 4096".split())
    torch.cuda.synchronize()
    P = prompt.shape[1]
    assert (count > 9).all() and (count < 1 + 9 * 6).any(), "some drafts stand, some do not"
    for n in held:
        assert n.tolist() == (count + P - 1).tolist()
    for b, n in enumerate(count.tolist()):
        assert (ids[b, :n] >= 0).all() and (ids[b, n:] == -1).all()
        text = torch.cat((prompt[b], ids[b, :n - 1])).unsqueeze(0)
        caches = target.caches(1, text.shape[1])
        none = torch.zeros(1, dtype=torch.int32, device=dev)
        logits = target(text, torch.arange(text.shape[1], device=dev).unsqueeze(0), caches, none)[0][0, P - 1:].float()
        best, scale = logits.max(1).values, logits.abs().max(1).values
        mine = logits.gather(1, ids[b, :n].unsqueeze(1)).squeeze(1)
        assert (mine >= best - scale / 16).all()


def test_eviction_bounds_the_cache(example, dev):
    """With eviction every fourth block a cache holds ``keep`` slots after it, and ids go on."""
    print("case kv4 example, eviction", flush=True)
    target, prompt, ids, count, held = example.main("--batch 4 --prompt 300 --rounds 8 --keep 100 --recent 20".split())
    torch.cuda.synchronize()
    for n in held:
        assert n.tolist() == [100] * 4
    assert (count > 8).all()
    for b, n in enumerate(count.tolist()):
        assert ((ids[b, :n] >= 0) & (ids[b, :n] < target.embed.shape[0])).all() and (ids[b, n:] == -1).all()
