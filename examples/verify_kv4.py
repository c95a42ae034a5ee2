"""Draft blocks and their verification over a 4-bit key/value cache, on synthetic weights.

The loop of code/dflash.py:560-670 with the target's cache held by ``KV4Cache``: a block
is drafted (``DeLSDraftStep``), its keys and values enter the cache of every layer
(``kv4_append``), its queries attend over context and block (``kv4_attention``), the
target's ids say how many drafts stand, the accepted rows' attention is added up per slot
(``kv4_weights``), rejected rows are cropped by going on from a shorter length, and once
a cache may hold more than ``keep`` slots the least attended ones go (``kv4_evict``).
Lengths, accepted counts and ids stay on the GPU throughout.

    python examples/verify_kv4.py --batch 4 --prompt 300 --rounds 12 --keep 256

The target has random weights but for its LM head, which gives the successor of a token
in a fixed random order unless attention says otherwise; the drafter's hidden states are
those successors, some of them wrong.  So some drafts stand and some do not.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import __graft_entry__  # noqa: E402

dels = __graft_entry__.load_package()


class Target:
    """A small decoder (attention layers and an LM head) whose context is one KV4Cache a layer."""

    def __init__(self, *, vocab=4096, hidden=512, layers=2, q_heads=8, kv_heads=2, head_dim=64, seed=0, device):
        g = torch.Generator().manual_seed(seed)
        def weight(*shape, std):
            return (torch.randn(*shape, generator=g) * std).bfloat16().to(device)
        self.q_heads, self.kv_heads, self.head_dim, self.device = q_heads, kv_heads, head_dim, device
        self.embed = weight(vocab, hidden, std=1.0)
        self.successor = torch.randperm(vocab, generator=g).to(device)
        self.lm_head = torch.empty_like(self.embed)
        self.lm_head[self.successor] = self.embed / hidden ** 0.5
        heads = q_heads + 2 * kv_heads
        self.qkv = [weight(heads * head_dim, hidden, std=hidden ** -0.5) for _ in range(layers)]
        self.out = [weight(hidden, q_heads * head_dim, std=(q_heads * head_dim) ** -0.5) for _ in range(layers)]
        self.freq = (10000.0 ** (-torch.arange(0, head_dim, 2) / head_dim)).to(device)

    def caches(self, batch, slots):
        return [dels.KV4Cache.allocate(batch, slots, self.kv_heads, self.head_dim, self.device) for _ in self.qkv]

    def _rotate(self, x, at):
        angle = (at.unsqueeze(-1) * self.freq).unsqueeze(2)
        a, b = x.float().chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1).bfloat16()

    def __call__(self, ids, positions, caches, lengths):
        """Logits of a block's rows, and (queries, lse) of each layer; the block enters the caches.

        ``positions`` are the rows' places in the text, ``lengths`` the slots the caches hold:
        they part ways once slots have been evicted.
        """
        B, T = ids.shape
        x, seen = self.embed[ids], []
        for cache, qkv, out in zip(caches, self.qkv, self.out):
            norm = torch.nn.functional.rms_norm(x.float(), x.shape[-1:]).bfloat16()
            rows = (norm.view(B * T, -1) @ qkv.t()).view(B, T, -1, self.head_dim)
            q, k, v = rows.split((self.q_heads, self.kv_heads, self.kv_heads), 2)
            q, k = self._rotate(q, positions), self._rotate(k, positions)
            dels.kv4_append(cache, k, v, lengths)
            o, lse = dels.kv4_attention(q, cache, lengths)
            seen.append((q, lse))
            x = x + 0.5 * (o.reshape(B * T, -1) @ out.t()).view(B, T, -1)
        return (x.view(B * T, -1) @ self.lm_head.t()).view(B, T, -1), seen


class Drafter:
    """Hidden states of a drafter that knows the order but errs, through ``DeLSDraftStep``."""

    def __init__(self, target, batch, k_draft, seed=1, noise=6.0):
        vocab, hidden = target.embed.shape
        torch.manual_seed(seed)
        holder = torch.nn.Module()
        holder.model, holder.lm_head = torch.nn.Module(), torch.nn.Linear(hidden, vocab, bias=False)
        holder.model.embed_tokens = torch.nn.Embedding(vocab, 64)
        head = dels.DeLSLocalHead(target_model=holder, vocab_size=vocab, embed_dim=64, gru_hidden_dim=128,
                                  low_rank_dim=64, lm_head_mode="direct_vocab", dtype=torch.bfloat16,
                                  device=target.device).to(target.device, torch.bfloat16)
        self.target, self.k, self.noise = target, k_draft, noise
        self.step = dels.DeLSDraftStep(local_head=head, lm_head_weight=target.lm_head, batch_size=batch,
                                       k_draft=k_draft, vocab_size=vocab, alpha_values=[0.1] * (k_draft - 1),
                                       beta_values=[0.0] * (k_draft - 1), baseline_logits=None,
                                       device=target.device)

    def __call__(self, last):
        ids = [last]
        for _ in range(self.k - 1):
            ids.append(self.target.successor[ids[-1]])
        hidden = self.target.embed[torch.stack(ids, 1)]
        return self.step(hidden + self.noise * torch.randn_like(hidden))


@torch.inference_mode()
def run(target, drafter, prompt, rounds, keep, recent, evict_every=4):
    """Greedy ids of a prompt's continuation: (ids, their numbers per sequence, slots held)."""
    B, P = prompt.shape
    dev, k = target.device, drafter.k
    # what a cache can hold: the prompt or what eviction leaves, and blocks until the next one
    caches = target.caches(B, max(P, keep) + evict_every * (k + 1))
    weights = [torch.zeros(B, c.kv_heads, c.slots, device=dev) for c in caches]
    held = [torch.zeros(B, dtype=torch.int32, device=dev) for _ in caches]

    at = torch.arange(P, device=dev).expand(B, P)
    logits, seen = target(prompt, at, caches, held[0])
    for cache, (q, lse), w, n in zip(caches, seen, weights, held):
        dels.kv4_weights(q, cache, n, lse, w, out=w)
    held = [n + P for n in held]
    last = dels.argmax_rows(logits[:, -1])[0]
    ids = torch.full((B, 1 + rounds * (k + 1)), -1, device=dev)
    ids[:, 0] = last
    count = torch.ones(B, dtype=torch.long, device=dev)

    for r in range(1, rounds + 1):
        drafts = drafter(last)
        block = torch.cat((last.unsqueeze(1), drafts), 1)
        at = (P - 1 + count).unsqueeze(1) + torch.arange(k + 1, device=dev)
        logits, seen = target(block, at, caches, held[0])
        best = dels.argmax_rows(logits.view(B * (k + 1), -1))[0].view(B, k + 1)
        right = (drafts == best[:, :-1]).long().cumprod(1).sum(1)
        rows = (right + 1).int()                     # the row that was given, and the drafts that stand
        for cache, (q, lse), w, n in zip(caches, seen, weights, held):
            dels.kv4_weights(q, cache, n, lse, w, rows, out=w)
        held = [n + rows for n in held]              # the other rows are cropped
        j = torch.arange(k + 1, device=dev).expand(B, -1)
        ids.scatter_(1, count.unsqueeze(1) + j, torch.where(j < rows.unsqueeze(1), best, -1))
        last = best.gather(1, right.unsqueeze(1)).squeeze(1)
        count = count + rows
        if r % evict_every == 0:
            for i, cache in enumerate(caches):
                held[i], weights[i], _ = dels.kv4_evict(cache, held[i], weights[i], keep, recent)
    return ids, count, held


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--rounds", type=int, default=12)
    ap.add_argument("--draft", type=int, default=7)
    ap.add_argument("--keep", type=int, default=256)
    ap.add_argument("--recent", type=int, default=64)
    a = ap.parse_args(argv)
    target = Target(device=torch.device("cuda:0"))
    drafter = Drafter(target, a.batch, a.draft)
    prompt = torch.randint(0, target.embed.shape[0], (a.batch, a.prompt),
                           generator=torch.Generator().manual_seed(2)).to(target.device)
    ids, count, held = run(target, drafter, prompt, a.rounds, a.keep, a.recent)
    print(f"{a.rounds} blocks of {a.draft} drafts: {[n - 1 for n in count.tolist()]} ids, "
          f"{held[0].tolist()} of {(count + a.prompt - 1).tolist()} slots held")
    return target, prompt, ids, count, held


if __name__ == "__main__":
    main()
