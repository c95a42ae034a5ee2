"""The measured calls of the 4-bit key/value cache: what writes it, reads it, attends over it and shrinks it.

A speculative-decoding server holds each sequence's keys and values in pages of
64 slots, four bits a value, and makes these calls around every draft block: the
block's keys and values are appended, the block's queries attend over context
and block, the weights that the accepted rows gave to each slot are added up,
and now and then the slots with the least weight are evicted.  Head counts and
head size are those of the Qwen3 heads that the benchmark uses (32 query heads
over 8 key/value heads of 128) or generic; a block is the benchmark's 16 tokens,
a prompt's chunk, or one token.

A page of one key/value head of D channels holds, in this order,
  * key codes, 64 rows of D/2 bytes, channel 2c in the low half of byte c;
  * key scales, 2^(byte - 127) per slot and 32 channels: slot
    32 s + 8 rh + 4 a + rl (s, a < 2, rh, rl < 4) of block m at byte
    64 m + 16 rh + 4 rl + 2 s + a;
  * value codes, 8 rows (one per 8 slots) of D little-endian words, slot
    8 g + i in bits 4 i .. 4 i + 3 of its channel's word in row g;
  * value scales, 64 bfloat16 numbers.
A code is sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6.
"""

from __future__ import annotations

import math

import torch

own = False          # whether run() makes the framework's calls or computes the plain form

DEV = "cuda:0"
PAGE = 64
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BIG = 3.0e38
SIXTH = 0.16666667163372040          # 1/6 in single precision


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # the 16 rows of a draft block of 8 sequences enter the cache: the server's usual write
        dict(name="append_block_b8", kind="append", B=8, T=16, H=8, D=128, ctx=2000, spread=0.75, dtype="bfloat16",
             heads_first=False, ragged=False),
        # prompts of up to 2039 tokens of four sequences, from a projection that lays heads before tokens
        dict(name="append_prompt_b4", kind="append", B=4, T=2039, H=8, D=128, ctx=0, spread=0.0, dtype="float16",
             heads_first=True, ragged=True),
        # one sequence, one token, a short context: the smallest call, where latency counts
        dict(name="attn_b1_t1", kind="attention", B=1, T=1, HQ=32, H=8, D=128, ctx=700, spread=0.0, dtype="bfloat16",
             block="causal", ragged=False, width=4096),
        # verification of a draft block of 16 for 8 sequences of uneven lengths
        dict(name="attn_b8_t16", kind="attention", B=8, T=16, HQ=32, H=8, D=128, ctx=4000, spread=0.875,
             dtype="bfloat16", block="causal", ragged=False, width=8192),
        # a tree of 33 drafted tokens, each seeing its own branch; five heads of 64 to each key/value head
        dict(name="attn_b5_tree33", kind="attention", B=5, T=33, HQ=20, H=4, D=64, ctx=1501, spread=0.5,
             dtype="float16", block="tree", ragged=False, width=2048),
        # one token each for 32 long conversations: the largest read of the cache
        dict(name="attn_b32_t1_16k", kind="attention", B=32, T=1, HQ=32, H=8, D=128, ctx=16300, spread=0.25,
             dtype="bfloat16", block="causal", ragged=False, width=16384),
        # a draft block over one very long document: few rows, the long axis has to be split
        dict(name="attn_b1_t16_131k", kind="attention", B=1, T=16, HQ=32, H=8, D=128, ctx=130900, spread=0.0,
             dtype="bfloat16", block="full", ragged=False, width=131072),
        # chunks of up to 512 prompt tokens over what is cached: bound by arithmetic
        dict(name="attn_b2_t512", kind="attention", B=2, T=512, HQ=32, H=8, D=128, ctx=3500, spread=0.5,
             dtype="bfloat16", block="causal", ragged=True, width=8192),
        # the weights that the accepted rows of 8 draft blocks gave to each slot
        dict(name="weights_b8_t16", kind="weights", B=8, T=16, HQ=32, H=8, D=128, ctx=4000, spread=0.875,
             dtype="bfloat16", block="causal", ragged=False, width=8192),
        # the same for single tokens of 32 long conversations
        dict(name="weights_b32_t1_16k", kind="weights", B=32, T=1, HQ=32, H=8, D=128, ctx=16300, spread=0.25,
             dtype="bfloat16", block="causal", ragged=False, width=16384),
        # one sequence past its budget by a few blocks: the smallest eviction
        dict(name="evict_b1", kind="evict", B=1, H=8, D=128, ctx=600, spread=0.0, width=1024, keep=512, recent=64),
        # 16 long conversations cut down to a quarter
        dict(name="evict_b16_16k", kind="evict", B=16, H=8, D=128, ctx=16300, spread=0.5, width=16384, keep=4096,
             recent=500),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another member of the listed families: sizes spread over their logarithm, odd ones among them."""
    kind = rng.choice(["append", "attention", "attention", "weights", "evict"])
    D = rng.choice([64, 128, 128])
    H = rng.choice([1, 2, 4, 8, 8])
    B = _log_uniform(rng, 1, 32)
    spread = rng.choice([0.0, 0.3, 0.9])
    if kind == "append":
        T = _log_uniform(rng, 1, 2039 if B <= 4 else 8000 // B)
        return dict(kind=kind, B=B, T=T, H=H, D=D, ctx=_log_uniform(rng, 1, 4000) - 1, spread=spread,
                    dtype=rng.choice(["float32", "bfloat16", "float16"]), heads_first=rng.random() < 0.5,
                    ragged=rng.random() < 0.5)
    ctx = _log_uniform(rng, 1, min(131000, 16300 * 32 // B))
    if kind == "evict":
        ctx = min(ctx, 16300)
        keep = max(1, int(ctx * rng.choice([0.25, 0.5, 0.9, 1.1])))
        return dict(kind=kind, B=min(B, 16), H=H, D=D, ctx=ctx, spread=spread, width=ctx + rng.randrange(1, 500),
                    keep=keep, recent=rng.choice([0, keep // 8, keep]))
    G = rng.choice([1, 2, 3, 4, 4, 5, 8])
    block = rng.choice(["causal", "causal", "full", "none", "tree"])
    T = rng.choice([1, 1, _log_uniform(rng, 2, 64), _log_uniform(rng, 2, 512)])
    T = min(T, 64 if block == "tree" else 512)
    # no more products than the largest listed case
    ctx = max(1, min(ctx, 2 * 4000 * 512 * 32 // (B * T * H * G)))
    return dict(kind=kind, B=B, T=T, HQ=H * G, H=H, D=D, ctx=ctx, spread=spread,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), block=block, ragged=rng.random() < 0.3,
                width=ctx + T + rng.randrange(1, 1 + ctx))


def _contexts(case):
    """Tokens that each sequence has cached before the call, in no order."""
    B, ctx = case["B"], case["ctx"]
    return [ctx - int(ctx * case["spread"] * b / max(B - 1, 1)) for b in range(B)]


def _valid(case):
    """Valid rows of each sequence's block (None: all of them)."""
    if not case["ragged"]:
        return None
    B, T = case["B"], case["T"]
    return [max(1, T - (T * b) // (2 * B)) for b in range(B)]


def _accepted(case):
    """Rows of each block that verification accepted."""
    valid = _valid(case) or [case["T"]] * case["B"]
    return [1 + (5 * b + 3) % n for b, n in enumerate(valid)]


def _slot_bytes(D):
    return D + D // 32 + 2


def work(case):
    kind, B, H, D = case["kind"], case["B"], case["H"], case["D"]
    if kind == "append":
        rows = sum(_valid(case) or [case["T"]] * B) * H
        size = 4 if case["dtype"] == "float32" else 2
        # the rows in, the cache out; then the cache in and the values out
        return dict(bytes=rows * 2 * (2 * D * size + _slot_bytes(D)), flops=rows * 2 * D * 10)
    ctx = _contexts(case)
    if kind == "evict":
        keep, recent = case["keep"], min(case["recent"], case["keep"])
        total = 0
        for n in ctx:
            total += 4 * n + 4 * case["width"] + 4 * keep
            if n > keep:
                above = n - keep                          # slots that must go or move
                stay = min(recent, above)
                moved = stay + (keep - recent) * (above - stay) / max(1, n - recent)
                total += int(moved) * 2 * _slot_bytes(D)
        return dict(bytes=H * total, flops=H * sum(ctx) * 8)
    T, HQ = case["T"], case["HQ"]
    valid = _valid(case) or [T] * B
    rows = valid if kind == "attention" else _accepted(case)
    block = case["block"]
    seen = [n + (0 if block == "none" else c) for n, c in zip(ctx, valid)]
    pairs = sum(r * n + (r * (r + 1) // 2 if block in ("causal", "tree") else r * c if block == "full" else 0)
                for r, n, c in zip(rows, ctx, valid)) * HQ
    if kind == "attention":
        return dict(bytes=H * _slot_bytes(D) * sum(seen) + sum(valid) * HQ * (4 * D + 4), flops=4 * pairs * D)
    return dict(bytes=H * (D // 2 + D // 32) * sum(seen) + sum(rows) * HQ * (2 * D + 4) +
                4 * H * (sum(ctx) + B * _slots(case)), flops=2 * pairs * D)


# ---- the cache, in elementary operations ---------------------------------------

def _slots(case):
    """Slots of a sequence's row in the table of pages."""
    return -(-max(case.get("width", 0), case["ctx"] + case.get("T", 0)) // PAGE) * PAGE


def _clean(x):
    x = x.float()
    return torch.where(x == x, x, torch.zeros_like(x)).clamp(-BIG, BIG)


def _codes(x, step):
    """Codes of x at this step (broadcast): the nearest of the eight magnitudes, ties to the even code."""
    a = x.abs()
    c = (a > 0.25 * step).to(torch.uint8)
    c += a >= 0.75 * step
    c += a > 1.25 * step
    c += a >= 1.75 * step
    c += a > 2.5 * step
    c += a >= 3.5 * step
    c += a > 5.0 * step
    return c + 8 * (x < 0).to(torch.uint8)


def _levels(codes):
    """The numbers that codes stand for, in single precision."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return table[codes.int()]


def _key_codes(k):
    """(codes, exponent bytes) of keys [..., D]: the smallest power of two whose 7-fold holds each 32 channels."""
    x = _clean(k).unflatten(-1, (-1, 32))
    bits = x.abs().amax(-1).view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7fffff) > 0x600000)).clamp(1, 252).to(torch.int32)
    return _codes(x, (e << 23).view(torch.float32)[..., None]).flatten(-2), e.to(torch.uint8)


def _value_codes(v):
    """(codes, bfloat16 scales) of values [..., D]: a sixth of the largest magnitude."""
    x = _clean(v)
    s = (x.abs().amax(-1) * SIXTH).to(torch.bfloat16).clamp(min=2.0 ** -126)
    return _codes(x, s.float()[..., None]), s


def _key_values(codes, e):
    return (_levels(codes).unflatten(-1, (-1, 32)) * (e.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _value_values(codes, s):
    return _levels(codes) * s.float()[..., None]


def _pack(kc, ke, vc, vs):
    """Pages [N, H, bytes] of codes [N, H, 64, D], exponent bytes [N, H, 64, D/32] and scales [N, H, 64]."""
    N, H, _, D = kc.shape
    k = (kc[..., 0::2] | (kc[..., 1::2] << 4)).reshape(N, H, -1)
    e = ke.reshape(N, H, 2, 4, 2, 4, D // 32).permute(0, 1, 6, 3, 5, 2, 4).reshape(N, H, -1)
    w = vc.view(N, H, 8, 4, 2, D)
    v = (w[..., 0, :] | (w[..., 1, :] << 4)).permute(0, 1, 2, 4, 3).reshape(N, H, -1)
    return torch.cat([k, e, v, vs.contiguous().view(torch.uint8).reshape(N, H, -1)], -1)


def _unpack(pages, D):
    """The reverse of _pack, of pages [..., bytes]: four tensors [..., 64, D or D/32 or none]."""
    lead = pages.shape[:-1]
    k, e, v, s = pages.split([32 * D, 2 * D, 32 * D, 128], -1)
    k = k.reshape(*lead, 64, D // 2)
    kc = torch.stack([k & 15, k >> 4], -1).flatten(-2)
    n = len(lead)
    e = e.reshape(*lead, D // 32, 4, 4, 2, 2).permute(*range(n), n + 3, n + 1, n + 4, n + 2, n).reshape(*lead, 64, -1)
    v = v.reshape(*lead, 8, D, 4).transpose(-1, -2)
    vc = torch.stack([v & 15, v >> 4], -2).reshape(*lead, 64, D)
    return kc, e, vc, s.contiguous().view(torch.bfloat16)


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys(shape, g):
    """Keys as attention layers have them: a few channels several times as wide as the others."""
    D = shape[-1]
    wide = torch.ones(D, device=DEV)
    wide[torch.randperm(D, generator=g, device=DEV)[:D // 16]] = 6.0
    return torch.randn(*shape, generator=g, device=DEV) * wide


def _source(case, seed):
    """Codes and scales of every slot that a sequence may use, [B, S, ...], drawn sequence by sequence."""
    g = _gen(seed)
    n = -(-(case["ctx"] + case.get("T", 0)) // PAGE) * PAGE
    parts = []
    for _ in range(case["B"]):
        shape = (case["H"], n, case["D"])
        parts.append((*_key_codes(_keys(shape, g)), *_value_codes(torch.randn(*shape, generator=g, device=DEV))))
    return [torch.stack(x) for x in zip(*parts)]           # [B, H, n, ...]


def _lengths(case, g):
    n = torch.tensor(_contexts(case), dtype=torch.int32, device=DEV)
    return n[torch.randperm(len(n), generator=g, device=DEV)]


def _pages(case, source, g):
    """Pages in the order in which a server hands them out, and each sequence's row of their numbers."""
    B, H = case["B"], case["H"]
    n = source[0].shape[2] // PAGE
    packed = _pack(*(x.unflatten(2, (n, PAGE)).transpose(1, 2).flatten(0, 1) for x in source))
    order = torch.randperm(B * n, generator=g, device=DEV)
    data = torch.empty_like(packed)
    data[order] = packed
    table = torch.zeros(B, _slots(case) // PAGE, dtype=torch.int32, device=DEV)
    table[:, :n] = order.view(B, n).int()
    return data, table


def _block_arg(case, g):
    """What the call takes for the block: a word, or for each row of a tree the bits of the rows that it sees."""
    if case["block"] != "tree":
        return case["block"]
    T = case["T"]
    bits = torch.zeros(case["B"], T, dtype=torch.int64)
    pick = torch.rand(case["B"], T, generator=g, device=DEV).cpu()
    for b in range(case["B"]):
        for t in range(T):
            up = int(bits[b, int(pick[b, t] * t)]) if t else 0
            here = up | (1 << t)
            bits[b, t] = here - (1 << 64) if here >= 1 << 63 else here
    return bits.to(DEV)


def _inputs(case, seed, want_cache=True):
    g = _gen(seed + 1)
    kind, B, H, D = case["kind"], case["B"], case["H"], case["D"]
    s = dict(case=case)
    s["lengths"] = _lengths(case, g)
    if kind == "evict":
        # weights of very uneven size, some slots that nothing ever attended to
        w = torch.exp(2.0 * torch.randn(B, H, _slots(case), generator=g, device=DEV))
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.05, torch.zeros_like(w), w)
    else:
        T = case["T"]
        valid = _valid(case)
        s["counts"] = None if valid is None else torch.tensor(valid, dtype=torch.int32, device=DEV)
    if kind == "append":
        shape = (B, H, T, D) if case["heads_first"] else (B, T, H, D)
        s["k"], s["v"] = (x.to(DTYPES[case["dtype"]]) for x in
                          (_keys(shape, g), torch.randn(*shape, generator=g, device=DEV)))
        if case["heads_first"]:
            s["k"], s["v"] = s["k"].transpose(1, 2), s["v"].transpose(1, 2)
    elif kind != "evict":
        s["q"] = torch.randn(B, T, case["HQ"], D, generator=g, device=DEV).to(DTYPES[case["dtype"]])
        s["block"] = _block_arg(case, g)
    if kind == "weights":
        s["accepted"] = torch.tensor(_accepted(case), dtype=torch.int32, device=DEV)
        s["weights"] = torch.rand(B, H, _slots(case), generator=g, device=DEV) * 4.0
    if want_cache:
        s["data"], s["table"] = _pages(case, _source(case, seed), g)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "weights":
        s["lse"] = _plain_attention(s)[1]
    if own:
        from __graft_entry__ import load_package

        s["pkg"] = load_package()
        s["cache"] = s["pkg"].KV4Cache(s["data"], s["table"], case["D"])
    return s


# ---- one pass --------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return _calls(s, kind)
    if kind == "append":
        return _plain_append(s)
    if kind == "attention":
        return dict(zip(("out", "lse"), _plain_attention(s)))
    return _plain_weights(s) if kind == "weights" else _plain_evict(s)


def _calls(s, kind):
    pkg, cache, case = s["pkg"], s["cache"], s["case"]
    if kind == "append":
        pkg.kv4_append(cache, s["k"], s["v"], s["lengths"], counts=s["counts"])
        k, v = pkg.kv4_read(cache, s["lengths"], case["T"], counts=s["counts"], dtype=s["k"].dtype)
        return dict(k=k, v=v)
    if kind == "attention":
        out, lse = pkg.kv4_attention(s["q"], cache, s["lengths"], block=s["block"], counts=s["counts"])
        return dict(out=out, lse=lse)
    if kind == "weights":
        return dict(weights=pkg.kv4_weights(s["q"], cache, s["lengths"], s["lse"], s["weights"], s["accepted"],
                                            block=s["block"], counts=s["counts"]))
    lengths, weights, source = pkg.kv4_evict(cache, s["lengths"], s["weights"], case["keep"], case["recent"])
    return dict(lengths=lengths, weights=weights, source=source, data=s["data"])


def _rows(s):
    """Whether each row of the block is valid, [B, T]."""
    T, B = s["case"]["T"], s["case"]["B"]
    t = torch.arange(T, device=DEV)
    if s["counts"] is None:
        return torch.ones(B, T, dtype=torch.bool, device=DEV)
    return t < s["counts"][:, None]


def _plain_append(s):
    """The values that the appended rows stand for in the cache."""
    keep = _rows(s)[:, :, None, None]
    k, v = _key_values(*_key_codes(s["k"])), _value_values(*_value_codes(s["v"]))
    return dict(k=torch.where(keep, k, torch.zeros_like(k)).to(s["k"].dtype),
                v=torch.where(keep, v, torch.zeros_like(v)).to(s["v"].dtype))


def _visible(s, n):
    """Which of n slots each row of the block sees, [B, T, n]."""
    B, T = s["case"]["B"], s["case"]["T"]
    j = torch.arange(n, device=DEV)
    own_slot = j - s["lengths"][:, None, None]                     # [B, 1, n], below 0: context
    t = torch.arange(T, device=DEV)[None, :, None]
    count = torch.full((B,), T, device=DEV) if s["counts"] is None else s["counts"]
    inside = own_slot < count[:, None, None]
    block = s["block"]
    if isinstance(block, torch.Tensor):
        seen = inside & (own_slot >= 0) & (((block[:, :, None] >> own_slot.clamp(0, 63)) & 1) == 1)
    elif block == "causal":
        seen = inside & (own_slot >= 0) & (own_slot <= t)
    elif block == "full":
        seen = inside & (own_slot >= 0)
    else:
        seen = torch.zeros_like(inside)
    return ((own_slot < 0) | seen) & _rows(s)[:, :, None]


def _grouped_scores(s, keys):
    """Scaled products [B, H, T, G, n] of the block's queries with keys [B, H, n, D]; -inf where a row does not see."""
    case = s["case"]
    B, T, H, D = case["B"], case["T"], case["H"], case["D"]
    G = case["HQ"] // H
    q = s["q"].float().view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = torch.matmul(q, keys.transpose(-1, -2).contiguous()).view(B, H, T, G, -1) / math.sqrt(D)
    return x.masked_fill_(~_visible(s, x.shape[-1])[:, None, :, None, :], -math.inf)


def _held(s):
    """The cache's rows of pages that hold anything, [B, H, pages, bytes]."""
    n = -(-(s["case"]["ctx"] + s["case"]["T"]) // PAGE)
    return s["data"][s["table"][:, :n].long()].transpose(1, 2)


def _plain_attention(s):
    case = s["case"]
    B, T, HQ, D = case["B"], case["T"], case["HQ"], case["D"]
    kc, ke, vc, vs = _unpack(_held(s), D)
    x = _grouped_scores(s, _key_values(kc, ke).flatten(2, 3))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _value_values(vc, vs).flatten(2, 3)).view(B, case["H"], T, -1, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log())[..., 0]
    return (o.permute(0, 2, 1, 3, 4).reshape(B, T, HQ, D).to(s["q"].dtype),
            lse.permute(0, 2, 1, 3).reshape(B, T, HQ))


def _plain_weights(s):
    case = s["case"]
    B, T, H = case["B"], case["T"], case["H"]
    kc, ke, _, _ = _unpack(_held(s), case["D"])
    x = _grouped_scores(s, _key_values(kc, ke).flatten(2, 3))
    lse = s["lse"].view(B, T, H, -1).permute(0, 2, 1, 3)[..., None]
    t = torch.arange(T, device=DEV)[None, :]
    counted = ((t < s["accepted"][:, None])[:, None, :, None, None]) & (lse > -math.inf)
    p = torch.where(counted, x.sub_(torch.where(lse > -math.inf, lse, torch.zeros_like(lse))).exp_(),
                    torch.zeros_like(x))
    j = torch.arange(s["weights"].shape[-1], device=DEV)
    new = torch.where(j < s["lengths"][:, None, None], s["weights"], torch.zeros_like(s["weights"]))
    new[..., :x.shape[-1]] += p.sum((2, 3))
    return dict(weights=new)


def _plain_evict(s):
    """Selection by a stable sort, movement of whole slots; the cache changes in place, as the framework's does."""
    case, w, n = s["case"], s["weights"], s["lengths"].long()[:, None, None]
    B, H, D, keep, S = case["B"], case["H"], case["D"], case["keep"], s["weights"].shape[-1]
    recent = min(case["recent"], keep)
    j = torch.arange(S, device=DEV).expand(B, H, S)
    # recent slots first, then by weight, slots past the end last; equal weights by slot
    key = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w)
    by_weight = key.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.where(j >= n, 2, torch.where(j >= n - recent, 0, 1)).gather(-1, by_weight)
    order = by_weight.gather(-1, rank.sort(dim=-1, stable=True).indices)
    place = torch.empty_like(order).scatter_(-1, order, j)         # each slot's place in that order
    kept = (place < keep) & (j < n)
    source = torch.where(j < n, j, -1)
    # holes below keep and kept slots from keep on, both in ascending order
    hole, mover = (~kept) & (j < keep) & (j < n), kept & (j >= keep)
    movers = torch.where(mover, j, S).sort(dim=-1).values
    nth = hole.long().cumsum(-1) - 1
    source = torch.where(hole, movers.gather(-1, nth.clamp(min=0)), source)[..., :keep]
    if source.shape[-1] < keep:                                    # a budget past the table: nothing to move
        source = torch.cat([source, source.new_full((B, H, keep - S), -1)], -1)
    new = torch.zeros_like(w)
    m = min(keep, S)
    new[..., :m] = torch.where(source[..., :m] >= 0, w.gather(-1, source[..., :m].clamp(min=0)),
                               torch.zeros_like(w[..., :m]))
    # the cache's bytes: moved as they are, so they are compared as bytes
    held = -(-case["ctx"] // PAGE)
    table = s["table"][:, :held].long()
    kc, ke, vc, vs = (x.flatten(2, 3) for x in _unpack(s["data"][table].transpose(1, 2), D))
    full = torch.arange(held * PAGE, device=DEV).expand(B, H, -1).clone()
    m = min(keep, held * PAGE)
    full[..., :m] = torch.where(hole[..., :m], source[..., :m], full[..., :m])
    take = lambda x: x.gather(2, full[..., None].expand_as(x))      # noqa: E731
    paged = lambda x: x.unflatten(2, (held, PAGE)).transpose(1, 2).flatten(0, 1)    # noqa: E731
    s["data"][table.flatten()] = _pack(paged(take(kc)), paged(take(ke)), paged(take(vc)),
                                       paged(vs.gather(2, full)))
    return dict(lengths=s["lengths"].clamp(max=keep), weights=new, source=source.int(), data=s["data"])


# ---- the same in 64 bits, from the definitions -------------------------------------

def _nearest(y):
    """|y| <= 6 rounded to the eight magnitudes: halves below 2, whole numbers below 4, even ones above."""
    a = y.abs().clamp(max=6.0)
    r = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round()))
    return r * y.sign()


def _exact_append(case, seed):
    s = _inputs(case, seed, want_cache=False)
    out = {}
    for name in ("k", "v"):
        x = s[name].double()
        if name == "k":
            y = x.unflatten(-1, (-1, 32))
            m, e = torch.frexp(y.abs().amax(-1, keepdim=True))      # amax = m 2^e, m in [1/2, 1)
            step = torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 3, e - 2))
            y = (_nearest(y / step) * step).flatten(-2)
        else:
            step = (x.abs().amax(-1, keepdim=True) * SIXTH).float().bfloat16().double()
            y = _nearest(x / step) * step
        for b, n in enumerate(_valid(case) or []):
            y[b, n:] = 0
        out[name] = y
    return out


def _decode64(codes):
    mag = codes & 7
    e, f = (mag >> 1).double(), (mag & 1).double()
    v = torch.where(mag < 2, 0.5 * f, torch.exp2(e - 1) * (1 + 0.5 * f))
    return torch.where(codes >= 8, -v, v)


def _exact_rows(case, s, b, keys, t):
    """Scores of row t of sequence b's block with keys [H, n, D], in 64 bits: [H, G, slots that it sees], and those."""
    n = int(s["lengths"][b])
    count = case["T"] if s["counts"] is None else int(s["counts"][b])
    if t >= count:
        return None, None
    block = s["block"]
    if isinstance(block, torch.Tensor):
        bits = int(block[b, t])
        own_slots = [i for i in range(count) if (bits >> i) & 1]
    else:
        own_slots = list(range({"causal": min(t + 1, count), "full": count, "none": 0}[block]))
    seen = torch.tensor(list(range(n)) + [n + i for i in own_slots], device=DEV, dtype=torch.long)
    q = s["q"][b, t].double().view(case["H"], -1, case["D"])
    return torch.bmm(q, keys[:, seen].transpose(1, 2).contiguous()) / math.sqrt(case["D"]), seen


def exact(case, seed):
    kind = case["kind"]
    if kind == "append":
        return _exact_append(case, seed)
    if kind == "evict":
        return None                                                # moved and selected, nothing computed
    B, T, H, HQ, D = case["B"], case["T"], case["H"], case["HQ"], case["D"]
    if B * T > 1100:
        return None
    s = _inputs(case, seed, want_cache=False)
    kc, ke, vc, vs = _source(case, seed)
    out = torch.zeros(B, T, HQ, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, T, HQ), -math.inf, dtype=torch.float64, device=DEV)
    given = prepare(case, seed)["lse"].double() if kind == "weights" else None
    if kind == "weights":
        w = s["weights"].double()
        for b in range(B):
            w[b, :, int(s["lengths"][b]):] = 0
    for b in range(B):
        keys = (_decode64(kc[b]).unflatten(-1, (-1, 32)) * torch.exp2(ke[b].double() - 127)[..., None]).flatten(-2)
        values = _decode64(vc[b]) * vs[b].double()[..., None]
        for t in range(T if kind == "attention" else int(s["accepted"][b])):
            x, seen = _exact_rows(case, s, b, keys, t)
            if x is None or not len(seen):
                continue
            if kind == "weights":
                w[b][:, seen] += (x - given[b, t].view(H, -1, 1)).exp().sum(1)
                continue
            top = x.amax(-1, keepdim=True)
            p = (x - top).exp()
            total = p.sum(-1, keepdim=True)
            out[b, t] = (torch.bmm(p, values[:, seen].contiguous()) / total).reshape(HQ, D)
            lse[b, t] = (top + total.log()).reshape(HQ)
    return dict(weights=w) if kind == "weights" else dict(out=out, lse=lse)
