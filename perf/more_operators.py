"""The measured calls of the 8-bit key/value cache: rows appended with their rotation, and attention over it.

A speculative-decoding server that finds four bits too few holds keys and values in
e4m3 with one power of two for each 32 tokens and head.  Around every draft block it
makes these calls: the block's queries and keys are rotated by their positions, its
keys and values are appended; the block's queries attend over context and block,
all of it or a sliding window with the first tokens of the context.  Head counts and
head size are those of the Qwen3 heads that the benchmark uses (32 query heads over
8 key/value heads of 128) or generic; a block is the benchmark's 16 tokens, a
prompt's chunk, or one token.

A page of one key/value head of D channels holds 64 slots, two blocks u of 32, in
this order:
  * key bytes (e4m3), channel 16 c + i of slot s of block u at byte
    32 D u + 512 c + 16 pos(s) + i, pos(s) = 8 (s % 16 / 4) + 4 (s / 16) + s % 4;
  * value bytes, channel c of slot 16 h + i of block u at byte 64 D + 32 D u + 16 D h + 16 c + i;
  * 8 bytes for each block: the keys' exponent e (2^(e - 127)), the values', two of 0,
    and a little-endian word with the bits of the slots that hold no finite row;
  * 112 bytes of nothing.
"""

from __future__ import annotations

import math

import torch

own = False          # whether run() makes the framework's calls or computes the plain form

DEV = "cuda:0"
PAGE, BLOCK = 64, 32
LOW, HIGH = 63, 191  # exponents that a block may have
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- cases -------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence enters the cache: the smallest call, where latency counts
        dict(name="append_b1_t1", kind="append", B=1, T=1, HQ=32, H=8, D=128, ctx=700, spread=0.0, dtype="bfloat16",
             rot=128, interleaved=False, heads_first=False, ragged=False),
        # the 16 rows of a draft block of 8 sequences: the server's usual write
        dict(name="append_block_b8", kind="append", B=8, T=16, HQ=32, H=8, D=128, ctx=2000, spread=0.75,
             dtype="bfloat16", rot=128, interleaved=False, heads_first=False, ragged=False),
        # prompts of up to 2039 tokens of four sequences, from projections that lay heads before tokens;
        # half of the channels are rotated, in neighbouring pairs
        dict(name="append_prompt_b4", kind="append", B=4, T=2039, HQ=32, H=8, D=128, ctx=0, spread=0.0,
             dtype="float16", rot=64, interleaved=True, heads_first=True, ragged=True),
        # one sequence, one token, a short context: latency again
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
        # draft blocks of 8 sequences that see a window of 1000 tokens and the first four
        dict(name="window_b8_t16", kind="attention", B=8, T=16, HQ=32, H=8, D=128, ctx=4000, spread=0.875,
             dtype="float16", block="causal", ragged=False, width=8192, window=1000, sinks=4),
        # one token each for 32 long conversations through a window of 4096
        dict(name="window_b32_t1_16k", kind="attention", B=32, T=1, HQ=32, H=8, D=128, ctx=16300, spread=0.25,
             dtype="bfloat16", block="causal", ragged=False, width=16384, window=4096, sinks=4),
        # a prompt of 4093 tokens through a window of 1024: most of the square is never looked at
        dict(name="window_prompt_b1", kind="attention", B=1, T=4093, HQ=32, H=8, D=128, ctx=75, spread=0.0,
             dtype="bfloat16", block="causal", ragged=False, width=4224, window=1024, sinks=4),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another member of the listed families: sizes spread over their logarithm, odd ones among them."""
    kind = rng.choice(["append", "attention", "attention"])
    D = rng.choice([64, 128, 128])
    H = rng.choice([1, 2, 4, 8, 8])
    G = rng.choice([1, 2, 3, 4, 4, 5, 8])
    B = _log_uniform(rng, 1, 32)
    spread = rng.choice([0.0, 0.3, 0.9])
    if kind == "append":
        T = _log_uniform(rng, 1, 2039 if B <= 4 else 8000 // B)
        return dict(kind=kind, B=B, T=T, HQ=H * G if G <= 5 else H, H=H, D=D, ctx=_log_uniform(rng, 1, 4000) - 1,
                    spread=spread, dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]),
                    rot=rng.choice([0, D // 2, D, D]), interleaved=rng.random() < 0.3,
                    heads_first=rng.random() < 0.5, ragged=rng.random() < 0.5)
    ctx = _log_uniform(rng, 1, min(131000, 16300 * 32 // B))
    block = rng.choice(["causal", "causal", "full", "none", "tree"])
    T = rng.choice([1, 1, _log_uniform(rng, 2, 64), _log_uniform(rng, 2, 2048)])
    T = min(T, 64 if block == "tree" else 2048)
    # no more products than the largest listed case
    ctx = max(1, min(ctx, 2 * 4000 * 512 * 32 // (B * T * H * G)))
    T = min(T, 2 * 4000 * 512 * 32 // (B * H * G * (ctx + T)) + 1)
    case = dict(kind=kind, B=B, T=T, HQ=H * G, H=H, D=D, ctx=ctx, spread=spread,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), block=block, ragged=rng.random() < 0.3,
                width=ctx + T + rng.randrange(1, 1 + ctx))
    if rng.random() < 0.4:
        case.update(window=_log_uniform(rng, 1, max(2, ctx + T)), sinks=rng.choice([0, 1, 4, 4, 64, 130]))
    return case


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


def work(case):
    B, H, HQ, D, T = case["B"], case["H"], case["HQ"], case["D"], case["T"]
    ctx, valid = _contexts(case), _valid(case) or [T] * B
    if case["kind"] == "append":
        size = 4 if case["dtype"] == "float32" else 2
        rows = sum(valid) * H
        # rows in and the cache out, the blocks' rows in and their values out; queries in and out
        held = sum(n % BLOCK + c for n, c in zip(ctx, valid)) * H
        turned = sum(valid) * HQ * 2 * D * size if case["rot"] else 0
        return dict(bytes=rows * 2 * D * (size + 1) + held * 2 * D * (1 + size) + turned,
                    flops=rows * 2 * D * 8 + (sum(valid) * (HQ + H) * case["rot"] * 3))
    block, window, sinks = case["block"], case.get("window"), case.get("sinks", 0)
    pairs = read = 0
    for n, c in zip(ctx, valid):
        # what row t sees ends at ends(t); a window leaves the sinks and its last tokens
        ends = [n + (0 if block == "none" else c if block == "full" else t + 1) for t in range(c)]
        starts = [0 if window is None else max(0, n + t - window + 1) for t in range(c)]
        pairs += sum(max(0, e - s) + min(s, sinks, e) for s, e in zip(starts, ends))
        top, low = max(ends), min(starts)
        read += max(0, top - low) + min(low, sinks, top)
    return dict(bytes=H * read * 2 * D + sum(valid) * HQ * (4 * D + 4), flops=4 * pairs * HQ * D)


# ---- the cache, in elementary operations ---------------------------------------

def _slots(case):
    """Slots of a sequence's row in the table of pages."""
    return -(-max(case.get("width", 0), case["ctx"] + case["T"]) // PAGE) * PAGE


def _exponents(top):
    """Bytes of the smallest powers of two whose 448-fold holds the magnitudes `top`."""
    bits = top.float().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000)).clamp(LOW, HIGH).to(torch.int32)


def _power(e):
    return (e.int() << 23).view(torch.float32)


def _codes(x, e):
    """e4m3 bytes of x over the powers of two e (broadcast)."""
    return (x.float() * _power(254 - e.int())).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, e):
    return codes.view(torch.float8_e4m3fn).float() * _power(e)


def _pack(kc, ke, vc, ve):
    """Pages [N, H, bytes] of bytes [N, H, 2, 32, D] and exponents [N, H, 2]; every row is finite."""
    N, H, _, _, D = kc.shape
    # slot 16 h + 4 a + q lies at 8 a + 4 h + q
    k = kc.reshape(N, H, 2, 2, 4, 4, D // 16, 16).permute(0, 1, 2, 6, 4, 3, 5, 7).reshape(N, H, -1)
    v = vc.reshape(N, H, 2, 2, 16, D).permute(0, 1, 2, 3, 5, 4).reshape(N, H, -1)
    head = torch.zeros(N, H, 128, dtype=torch.uint8, device=kc.device)
    head[..., 0:16:8], head[..., 1:16:8] = ke.to(torch.uint8), ve.to(torch.uint8)
    return torch.cat([k, v, head], -1)


def _unpack(pages, D):
    """The reverse of _pack, of pages [..., bytes]: bytes [..., 2, 32, D], exponents [..., 2], twice."""
    lead = pages.shape[:-1]
    n = len(lead)
    k, v, head = pages.split([64 * D, 64 * D, 128], -1)
    k = k.reshape(*lead, 2, D // 16, 4, 2, 4, 16).permute(*range(n + 1), n + 3, n + 2, n + 4, n + 1, n + 5)
    v = v.reshape(*lead, 2, 2, D, 16).permute(*range(n + 1), n + 1, n + 3, n + 2)
    return (k.reshape(*lead, 2, BLOCK, D), head[..., 0:16:8], v.reshape(*lead, 2, BLOCK, D), head[..., 1:16:8])


# ---- inputs --------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys(shape, g):
    """Keys as attention layers have them: a few channels several times as wide as the others."""
    D = shape[-1]
    wide = torch.ones(D, device=DEV)
    wide[torch.randperm(D, generator=g, device=DEV)[:D // 16]] = 6.0
    return torch.randn(*shape, generator=g, device=DEV) * wide


def _quantised(x):
    """(bytes, exponents) of rows [H, n, D], 32 of them to a block."""
    x = x.unflatten(1, (-1, BLOCK))
    e = _exponents(x.abs().amax((-2, -1)))
    return _codes(x, e[..., None, None]), e


def _source(case, seed):
    """Bytes and exponents of every block that a sequence may use, [B, H, blocks, ...], sequence by sequence."""
    g = _gen(seed)
    n = -(-(case["ctx"] + case["T"]) // PAGE) * PAGE
    parts = []
    for _ in range(case["B"]):
        shape = (case["H"], n, case["D"])
        parts.append((*_quantised(_keys(shape, g)), *_quantised(torch.randn(*shape, generator=g, device=DEV))))
    return [torch.stack(x) for x in zip(*parts)]


def _lengths(case, g):
    n = torch.tensor(_contexts(case), dtype=torch.int32, device=DEV)
    return n[torch.randperm(len(n), generator=g, device=DEV)]


def _pages(case, source, g):
    """Pages in the order in which a server hands them out, and each sequence's row of their numbers."""
    B = case["B"]
    n = source[0].shape[2] // 2
    packed = _pack(*(x.unflatten(2, (n, 2)).transpose(1, 2).flatten(0, 1) for x in source))
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


def _tables(case):
    """Cosines and sines of every position, single precision, the angles in 64 bits."""
    half = case["rot"] // 2
    p = torch.arange(case["ctx"] + case["T"], dtype=torch.float64, device=DEV)
    angle = p[:, None] * 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    return angle.cos().float(), angle.sin().float()


def _inputs(case, seed, want_cache=True):
    g = _gen(seed + 1)
    B, H, D, T = case["B"], case["H"], case["D"], case["T"]
    s = dict(case=case)
    s["lengths"] = _lengths(case, g)
    valid = _valid(case)
    s["counts"] = None if valid is None else torch.tensor(valid, dtype=torch.int32, device=DEV)
    if case["kind"] == "append":
        def shape(h):
            return (B, h, T, D) if case["heads_first"] else (B, T, h, D)

        made = (_keys(shape(H), g), torch.randn(*shape(H), generator=g, device=DEV),
                torch.randn(*shape(case["HQ"]), generator=g, device=DEV))
        s["k"], s["v"], s["q"] = (x.to(DTYPES[case["dtype"]]).transpose(1, 2) if case["heads_first"] else
                                  x.to(DTYPES[case["dtype"]]) for x in made)
        s["cos"], s["sin"] = _tables(case) if case["rot"] else (None, None)
        # the blocks that the rows fall into are read back from their first slot
        s["starts"] = s["lengths"] // BLOCK * BLOCK
        s["held"] = s["lengths"] - s["starts"] + (T if valid is None else s["counts"])
    else:
        s["q"] = torch.randn(B, T, case["HQ"], D, generator=g, device=DEV).to(DTYPES[case["dtype"]])
        s["block"] = _block_arg(case, g)
    if want_cache:
        s["data"], s["table"] = _pages(case, _source(case, seed), g)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from __graft_entry__ import load_package

        s["pkg"] = load_package()
        s["cache"] = s["pkg"].KV8Cache(s["data"], s["table"], case["D"])
        if case["kind"] == "append":
            s["rotary"] = s["pkg"].RotaryTable(s["cos"], s["sin"], case["interleaved"]) if case["rot"] else None
    return s


# ---- one pass --------------------------------------------------------------------

def run(s):
    append = s["case"]["kind"] == "append"
    if own:
        return _call_append(s) if append else _call_attention(s)
    return _plain_append(s) if append else _plain_attention(s)


def _call_append(s):
    pkg, cache, case = s["pkg"], s["cache"], s["case"]
    if s["rotary"] is None:
        pkg.kv8_append(cache, s["k"], s["v"], s["lengths"], counts=s["counts"])
        q = None
    else:
        q = pkg.kv8_append(cache, s["k"], s["v"], s["lengths"], counts=s["counts"], rotary=s["rotary"], q=s["q"])
    k, v = pkg.kv8_read(cache, s["starts"], case["T"] + BLOCK - 1, counts=s["held"], dtype=s["k"].dtype)
    return dict(k=k, v=v) if q is None else dict(k=k, v=v, q=q)


def _call_attention(s):
    out, lse = s["pkg"].kv8_attention(s["q"], s["cache"], s["lengths"], block=s["block"], counts=s["counts"],
                                      window=s["case"].get("window"), sinks=s["case"].get("sinks", 0))
    return dict(out=out, lse=lse)


def _rows(s):
    """Whether each row of the block is valid, [B, T]."""
    T, B = s["case"]["T"], s["case"]["B"]
    t = torch.arange(T, device=DEV)
    if s["counts"] is None:
        return torch.ones(B, T, dtype=torch.bool, device=DEV)
    return t < s["counts"][:, None]


def _turned(s, x):
    """Rows [B, T, heads, D] rotated by the angles of their positions, in single precision."""
    case, x = s["case"], x.float()
    rot = case["rot"]
    if not rot:
        return x
    at = (s["lengths"].long()[:, None] + torch.arange(case["T"], device=DEV)).clamp(max=s["cos"].shape[0] - 1)
    c, d = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    y = x.clone()
    first, second = a * c - b * d, b * c + a * d
    if case["interleaved"]:
        y[..., 0:rot:2], y[..., 1:rot:2] = first, second
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = first, second
    return y


def _blocks_with(s, x):
    """(rows [B, H, blocks, 32, D] from each sequence's first block on, which of them are new)."""
    case = s["case"]
    B, T = case["B"], case["T"]
    n = -(-(T + BLOCK - 1) // BLOCK)
    skip = (s["lengths"] % BLOCK).long()
    rows = torch.zeros(B, n * BLOCK, case["H"], case["D"], device=DEV)
    new = torch.zeros(B, n * BLOCK, dtype=torch.bool, device=DEV)
    at = skip[:, None] + torch.arange(T, device=DEV)
    rows.scatter_(1, at[:, :, None, None].expand(-1, -1, case["H"], case["D"]), x)
    new.scatter_(1, at, _rows(s))
    return rows.unflatten(1, (n, BLOCK)).permute(0, 3, 1, 2, 4), new.unflatten(1, (n, BLOCK))[:, None]


def _joined(old_codes, old_e, x, new, kept):
    """Blocks of kept old rows and new rows under one exponent each: (bytes, exponents)."""
    top = torch.where(new[..., None], x, torch.zeros_like(x)).abs().amax((-2, -1))
    e = torch.where(kept.any(-1), torch.maximum(_exponents(top), old_e.int()), _exponents(top))
    moved = (old_codes.view(torch.float8_e4m3fn).float() * _power(127 + old_e.int() - e)[..., None, None])
    codes = torch.where(new[..., None], _codes(x, e[..., None, None]),
                        moved.to(torch.float8_e4m3fn).view(torch.uint8))
    return torch.where((kept | new)[..., None], codes, torch.zeros_like(codes)), e


def _plain_append(s):
    """The cache changes in place, as the framework's does; the values that the touched blocks' rows stand for."""
    case = s["case"]
    B, T, D = case["B"], case["T"], case["D"]
    first = (s["starts"] // BLOCK).long()                          # blocks; an odd one is a page's second
    k, new = _blocks_with(s, _turned(s, s["k"]))
    v, _ = _blocks_with(s, s["v"].float())
    n = new.shape[2]
    pages = (n + 2) // 2
    held = s["table"].shape[1]
    at = (first[:, None] // 2 + torch.arange(pages, device=DEV)).clamp(max=held - 1)
    page = s["table"].gather(1, at).long()                         # [B, pages]
    kc, ke, vc, ve = (x.transpose(1, 2).flatten(2, 3) for x in _unpack(s["data"][page], D))     # [B, H, blocks, ...]
    index = (first % 2)[:, None] + torch.arange(n, device=DEV)     # the rows' blocks among those
    take = index[:, None].expand(-1, case["H"], -1)
    pick = take[..., None, None].expand(-1, -1, -1, BLOCK, D)
    j = (torch.arange(n * BLOCK, device=DEV)).view(n, BLOCK)
    kept = (j < (s["lengths"] % BLOCK)[:, None, None])[:, None]
    knew, e1 = _joined(kc.gather(2, pick), ke.gather(2, take), k, new, kept)
    vnew, e2 = _joined(vc.gather(2, pick), ve.gather(2, take), v, new, kept)
    touched = new.any(-1).expand(-1, case["H"], -1)
    ones = touched[..., None, None]
    kc = kc.scatter(2, pick, torch.where(ones, knew, kc.gather(2, pick)))
    vc = vc.scatter(2, pick, torch.where(ones, vnew, vc.gather(2, pick)))
    ke = ke.scatter(2, take, torch.where(touched, e1.to(torch.uint8), ke.gather(2, take)))
    ve = ve.scatter(2, take, torch.where(touched, e2.to(torch.uint8), ve.gather(2, take)))
    packed = _pack(*(x.unflatten(2, (pages, 2)).transpose(1, 2).flatten(0, 1) for x in (kc, ke, vc, ve)))
    # pages past a sequence's own (the clamped column) are not written
    real = (first[:, None] // 2 + torch.arange(pages, device=DEV)) * PAGE < s["lengths"][:, None] + T
    real = real & (first[:, None] // 2 + torch.arange(pages, device=DEV) < held)
    s["data"][page.flatten()[real.flatten()]] = packed[real.flatten()]
    shown = (torch.arange(T + BLOCK - 1, device=DEV) < s["held"][:, None])[:, :, None, None]
    out = {}
    for name, codes, e in (("k", knew, e1), ("v", vnew, e2)):
        x = _values(codes, e[..., None, None]).flatten(2, 3).transpose(1, 2)[:, :T + BLOCK - 1]
        out[name] = torch.where(shown, x, torch.zeros_like(x)).to(s["k"].dtype)
    if case["rot"]:
        q = _turned(s, s["q"])
        out["q"] = torch.where(_rows(s)[:, :, None, None], q, torch.zeros_like(q)).to(s["q"].dtype)
    return out


def _visible(s, n):
    """Which of n slots each row of the block sees, [B, T, n]."""
    case = s["case"]
    B, T = case["B"], case["T"]
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
    seen = (own_slot < 0) | seen
    if case.get("window") is not None:
        seen = seen & ((own_slot > t - case["window"]) | (j < case["sinks"]))
    return seen & _rows(s)[:, :, None]


def _plain_attention(s):
    case = s["case"]
    B, T, H, HQ, D = case["B"], case["T"], case["H"], case["HQ"], case["D"]
    G = HQ // H
    n = -(-(case["ctx"] + T) // PAGE)
    kc, ke, vc, ve = _unpack(s["data"][s["table"][:, :n].long()].transpose(1, 2), D)      # [B, H, pages, 2, ...]
    keys = _values(kc, ke[..., None, None]).flatten(2, 4)
    q = s["q"].float().view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D)
    x = torch.matmul(q, keys.transpose(-1, -2).contiguous()).view(B, H, T, G, -1) / math.sqrt(D)
    x = x.masked_fill_(~_visible(s, x.shape[-1])[:, None, :, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _values(vc, ve[..., None, None]).flatten(2, 4)).view(B, H, T, G, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log())[..., 0]
    return dict(out=o.permute(0, 2, 1, 3, 4).reshape(B, T, HQ, D).to(s["q"].dtype),
                lse=lse.permute(0, 2, 1, 3).reshape(B, T, HQ))


# ---- the same in 64 bits, from the definitions -------------------------------------

def _grid(y):
    """Numbers of magnitude up to 448 rounded to e4m3: three bits after the first, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(y)                                          # y = m 2^e, m in [1/2, 1)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (y / step).round() * step


def _decode64(codes):
    e, f = ((codes >> 3) & 15).double(), (codes & 7).double()
    v = torch.where(e > 0, torch.exp2(e - 7) * (1 + f / 8), f * 2.0 ** -9)
    return torch.where(codes >= 128, -v, v)


def _least(top):
    """Exponents of the least powers of two (from 2^-64 on) whose 448-fold is at least `top`."""
    m, e = torch.frexp(top)
    return torch.where(m <= 0.875, e - 9, e - 8).clamp(LOW - 127, HIGH - 127).double()


def _exact_turn(s, x):
    """Rotation with products and sums rounded to single precision, as the operator defines them."""
    rot = s["case"]["rot"]
    x = x.double().clone()
    if not rot:
        return x
    for b, n in enumerate(s["lengths"].tolist()):
        c, d = (t[n:n + x.shape[1], None].double() for t in (s["cos"], s["sin"]))
        i = torch.arange(rot // 2, device=DEV)
        i, j = (2 * i, 2 * i + 1) if s["case"]["interleaved"] else (i, i + rot // 2)
        u, w = x[b][..., i].clone(), x[b][..., j].clone()
        single = lambda y: y.float().double()                       # noqa: E731
        x[b][..., i] = single(single(u * c) - single(w * d))
        x[b][..., j] = single(single(w * c) + single(u * d))
    return x


def _exact_append(case, seed):
    s = _inputs(case, seed, want_cache=False)
    source = _source(case, seed)
    B, T = case["B"], case["T"]
    out = {}
    for name, codes, e in (("k", *source[:2]), ("v", *source[2:])):
        x = _exact_turn(s, s[name]) if name == "k" else s[name].double()
        y = torch.zeros(B, T + BLOCK - 1, case["H"], case["D"], dtype=torch.float64, device=DEV)
        for b in range(B):
            n, start = int(s["lengths"][b]), int(s["starts"][b])
            count = T if s["counts"] is None else int(s["counts"][b])
            for first in range(start, n + count, BLOCK):
                lo, hi = max(first, n), min(first + BLOCK, n + count)
                rows = x[b, lo - n:hi - n].transpose(0, 1)          # [H, rows, D]
                scale = _least(rows.abs().amax((1, 2)))
                if first < n:
                    was = e[b, :, first // BLOCK].double() - 127
                    scale = torch.maximum(scale, was)
                    old = _decode64(codes[b, :, first // BLOCK, :n - first])
                    step = torch.exp2(was - scale)[:, None, None]
                    kept = _grid(old * step) * torch.exp2(scale)[:, None, None]
                    y[b, first - start:n - start] = kept.transpose(0, 1)
                unit = torch.exp2(scale)[:, None, None]
                y[b, lo - start:hi - start] = (_grid(rows / unit) * unit).transpose(0, 1)
        out[name] = y
    if case["rot"]:
        out["q"] = _exact_turn(s, s["q"])
        for b, c in enumerate(_valid(case) or []):
            out["q"][b, c:] = 0
    return out


def exact(case, seed):
    if case["kind"] == "append":
        return _exact_append(case, seed)
    B, T, H, HQ, D = case["B"], case["T"], case["H"], case["HQ"], case["D"]
    s = _inputs(case, seed, want_cache=False)
    kc, ke, vc, ve = _source(case, seed)
    out = torch.zeros(B, T, HQ, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, T, HQ), -math.inf, dtype=torch.float64, device=DEV)
    window, sinks = case.get("window"), case.get("sinks", 0)
    for b in range(B):
        n = int(s["lengths"][b])
        count = T if s["counts"] is None else int(s["counts"][b])
        j = torch.arange(n + count, device=DEV)
        t = torch.arange(count, device=DEV)[:, None]
        if isinstance(s["block"], torch.Tensor):
            bits = s["block"][b, :count, None] >> (j - n).clamp(0, 63)
            see = (j < n) | ((bits & 1) == 1)
        else:
            see = j < n + {"causal": 1 + t, "full": 0 * t + count, "none": 0 * t}[s["block"]]
        if window is not None:
            see = see & ((j >= n + t - window + 1) | (j < sinks))
        some = see.any(1)
        for h in range(H):
            keys = (_decode64(kc[b, h]) * torch.exp2(ke[b, h].double() - 127)[:, None, None]).flatten(0, 1)[:n + count]
            vals = (_decode64(vc[b, h]) * torch.exp2(ve[b, h].double() - 127)[:, None, None]).flatten(0, 1)[:n + count]
            for hq in range(h * (HQ // H), (h + 1) * (HQ // H)):
                x = s["q"][b, :count, hq].double() @ keys.t() / math.sqrt(D)
                x = x.masked_fill(~see, -math.inf)
                top = x.amax(1, keepdim=True).clamp(min=-1e300)
                p = (x - top).exp()
                total = p.sum(1, keepdim=True)
                out[b, :count, hq] = (p @ vals / total).masked_fill(~some[:, None], 0.0)
                lse[b, :count, hq] = (top + total.log())[:, 0].masked_fill(~some, -math.inf)
    return dict(out=out, lse=lse)
