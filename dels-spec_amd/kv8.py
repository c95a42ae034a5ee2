"""Key/value cache held in 8 bits, rows rotated on their way into it, and attention over it (gfx950 kernels).

The target's side of a draft block's verification (code/dflash.py:637-651) for whom
four bits (``kv4``) are too few: keys and values are e4m3 numbers under one power of
two for each 32 slots and head, in pages of 64 slots (include/dels.h describes one).
Lengths live on the GPU and no call reads them back, so every call can be captured into
a graph; workspaces are as in ``kv4``.

  * ``kv8_append``    -- a block's rows into the cache, keys and queries rotated by their positions
  * ``kv8_read``      -- the values that slots of the cache stand for
  * ``kv8_attention`` -- attention of a block's rows, one token or a prompt's chunk, over all they
    may see or through a sliding window that leaves a few first slots visible

A length is the number of slots a sequence holds *before* the block, in all calls
alike: row ``t`` of a block lies in slot ``lengths[b] + t``.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .kv4 import (_Q_DTYPES, HEAD_DIMS, Block, PagedCache, _block_args, _capturing, _elsewhere, _own_workspace,
                  _require_cache, _require_ints, _require_lse, _require_rows, _row_stride)
from .ops import _DTYPES, _WORKSPACES, _require_cuda, _stream_ptr

BLOCK = 32             # slots that share a scale
_FAR = 1 << 40         # past every slot


def page_bytes(head_dim: int) -> int:
    """Bytes of one key/value head's page of 64 slots."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    return 128 * head_dim + 128


class KV8Cache(PagedCache):
    """Pages of an 8-bit key/value cache and the table that hands them out (``PagedCache`` says how)."""

    bits = 8
    page_bytes = staticmethod(page_bytes)


class RotaryTable:
    """Cosines and sines of positions, by which ``kv8_append`` rotates keys and queries.

    ``cos``, ``sin`` fp32 ``[positions, channels / 2]`` on the GPU, unit column stride and one
    row stride, rows 16-byte aligned; ``channels`` (a multiple of 16, at most the head's)
    are rotated, the others kept.  Pair ``i`` is channels ``i`` and ``i + channels / 2``,
    or ``2 i`` and ``2 i + 1`` where ``interleaved``: ``(a, b)`` becomes ``(a c - b s, b c + a s)``.
    The table keeps both tensors.
    """

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False):
        for t, name in ((cos, "cos"), (sin, "sin")):
            _require_cuda(t, name)
            if t.dtype != torch.float32 or t.dim() != 2:
                raise ValueError(f"{name} must be float32 [positions, channels / 2], got {t.dtype} {tuple(t.shape)}")
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError(f"{name} must have unit column stride")
        if cos.shape != sin.shape or cos.device != sin.device:
            raise ValueError("cos and sin must have one shape and device")
        if cos.shape[1] < 8 or cos.shape[1] % 8:
            raise ValueError(f"rotated channels must be a multiple of 16, got {2 * cos.shape[1]}")
        strides = [_row_stride(t, t.shape[1], n) for t, n in ((cos, "cos"), (sin, "sin"))]
        if strides[0] != strides[1]:
            raise ValueError("cos and sin must have one row stride")
        self.cos, self.sin = cos, sin
        self.channels = 2 * int(cos.shape[1])
        self.interleaved = bool(interleaved)
        self._index = cos.get_device()
        self._params = _lib.RotaryParams(cos.data_ptr(), sin.data_ptr(), strides[0], cos.shape[0], self.channels,
                                         int(self.interleaved))
        self._ref = ctypes.byref(self._params)


# the current GPU, without the wrapper's check that there is one
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _elsewhere_current(cache: PagedCache) -> bool:
    """Whether the current GPU is not the cache's: then it is made so for the call."""
    return cache._index >= 0 and _current_device() != cache._index


def _require_pair(k: torch.Tensor, v: torch.Tensor, cache: PagedCache) -> tuple:
    """(pointer, strides) of keys and values that are alike."""
    kp = _require_rows(k, cache, cache.kv_heads, "k", _DTYPES)
    if not isinstance(v, torch.Tensor) or v.get_device() != cache._index:
        _elsewhere(v, cache, "v")
    if v.dtype != k.dtype or v.shape != k.shape:
        _require_rows(v, cache, cache.kv_heads, "v", _DTYPES)
        raise ValueError("k and v must have one shape and dtype")
    if v.stride() == k.stride():
        return kp, (v.data_ptr(), *kp[1:])
    return kp, _require_rows(v, cache, cache.kv_heads, "v", _DTYPES)


_NO_ROWS = (None, 0, 0, 0)


def _position_args(positions: torch.Tensor, cache: PagedCache, T: int) -> tuple[int, int]:
    """(pointer, row stride) of int32 [batch, T] positions."""
    if not isinstance(positions, torch.Tensor) or positions.get_device() != cache._index:
        _elsewhere(positions, cache, "positions")
    if positions.dtype != torch.int32 or positions.shape != (cache.batch, T):
        raise ValueError(f"positions must be int32 [{cache.batch}, {T}], got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    if T > 1 and positions.stride(1) != 1:
        raise ValueError("positions must have unit column stride")
    return positions.data_ptr(), _row_stride(positions, T, "positions")


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, *,
               counts: Optional[torch.Tensor] = None, rotary: Optional[RotaryTable] = None,
               positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write rows ``t < counts[b]`` (None: all) of ``k`` and ``v`` into slots ``lengths[b] + t``.

    ``k``, ``v`` ``[batch, T, kv_heads, head_dim]`` fp32, bf16 or fp16, any strides that
    keep rows 16-byte aligned.  With a ``rotary`` table, keys are rotated by the angles of
    their positions, ``positions`` int32 ``[batch, T]`` or else ``lengths[b] + t``, in fp32, every
    product and sum rounded; so are ``q`` ``[batch, T, q_heads, head_dim]`` (``k``'s dtype), which
    go to ``q_out`` (``q`` itself, say; None: a new tensor), rounded to their type: that is returned,
    its rows from ``counts[b]`` on 0.

    A block of 32 slots has one exponent for its keys and one for its values: the smallest
    that holds its new rows, or that of the rows before them in the block if it is larger (rows
    that were rejected leave it as they made it); if it is smaller, those rows are rounded again.
    A row of which something is NaN, infinite or over 448 * 2^64, or whose position the table
    does not have, reads as NaN and gives scores of NaN, and takes no part in the exponents; a query
    at such a position has NaN in its rotated channels.
    ``lengths`` is not changed; rows past the table's slots are dropped.
    """
    _require_cache(cache, 8)
    if _elsewhere_current(cache):
        with torch.cuda.device(cache._index):
            return kv8_append(cache, k, v, lengths, counts=counts, rotary=rotary, positions=positions, q=q,
                              q_out=q_out)
    kp, vp = _require_pair(k, v, cache)
    T = k.shape[1]
    lp, cp = _require_ints(lengths, cache, "lengths"), _require_ints(counts, cache, "counts")
    if rotary is None and (positions is not None or q is not None):
        raise ValueError("positions and q are for a rotary table")
    if q is None and q_out is not None:
        raise ValueError("q_out is for q")
    ref, qp, op, heads, pp, ldp = None, _NO_ROWS, _NO_ROWS, 0, None, 0
    if rotary is not None:
        if rotary._index != cache._index:
            raise ValueError(f"the rotary table is on {rotary.cos.device}, the cache on {cache.device}")
        if rotary.channels > cache.head_dim:
            raise ValueError(f"{rotary.channels} rotated channels, heads of {cache.head_dim}")
        ref = rotary._ref
        if positions is not None:
            pp, ldp = _position_args(positions, cache, T)
    if q is not None:
        qp = _require_rows(q, cache, None, "q", (k.dtype,))
        shape = q.shape
        heads = shape[2]
        if shape[1] != T or heads < 1 or heads % cache.kv_heads:
            raise ValueError(f"q must be [{cache.batch}, {T}, a multiple of {cache.kv_heads}, {cache.head_dim}], got "
                             f"{tuple(shape)}")
        if q_out is None:
            q_out = torch.empty(shape, dtype=q.dtype, device=cache.device)
            D = cache.head_dim
            op = (q_out.data_ptr(), T * heads * D, heads * D, D)
        elif q_out.shape != shape:
            raise ValueError(f"q_out must be {tuple(shape)}, got {tuple(q_out.shape)}")
        else:
            op = _require_rows(q_out, cache, heads, "q_out", (q.dtype,))
    _lib.check(_lib.load().dels_kv8_append(cache._ref, *kp, *vp, _DTYPES[k.dtype], lp, cp, T, ref, pp, ldp, *qp,
                                           heads, *op, _stream_ptr(cache.device)), "dels_kv8_append")
    return q_out


def kv8_read(cache: KV8Cache, starts: torch.Tensor, T: int, *, counts: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys (as they were rotated) and values that slots ``starts[b] + t``, ``t < T``, stand for.

    Returns ``(k, v)``, each ``[batch, T, kv_heads, head_dim]`` of ``dtype``; zeros from
    ``counts[b]`` on (None: none) and past the table's slots, NaN for rows that were not finite.
    """
    _require_cache(cache, 8)
    if _elsewhere_current(cache):
        with torch.cuda.device(cache._index):
            return kv8_read(cache, starts, T, counts=counts, dtype=dtype)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype {dtype} not supported")
    sp, cp = _require_ints(starts, cache, "starts"), _require_ints(counts, cache, "counts")
    k = torch.empty(cache.batch, T, cache.kv_heads, cache.head_dim, dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    _lib.check(_lib.load().dels_kv8_read(cache._ref, sp, cp, T, k.data_ptr(), v.data_ptr(), _DTYPES[dtype],
                                         _stream_ptr(cache.device)), "dels_kv8_read")
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, lengths: torch.Tensor, *, block: Block = "causal",
                  counts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  window: Optional[int] = None, sinks: int = 0, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                  positions: Optional[torch.Tensor] = None,
                  weight_parts: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of a block's rows over their sequences' context and the block itself.

    ``q`` ``[batch, T, q_heads, head_dim]`` bf16 or fp16, ``q_heads`` a multiple of the
    cache's heads.  Every row sees slots ``[0, lengths[b])``; of the block's own slots
    (which ``kv8_append`` wrote) ``block`` says which: ``"causal"``, ``"full"``, ``"none"``, or
    an int64 ``[batch, T]`` of bits, bit ``i`` of row ``t`` for slot ``lengths[b] + i`` (a tree of
    drafts; T at most 64; expanded where all sequences have one tree).  With a ``window``,
    row ``t`` sees of these only the slots from ``lengths[b] + t - window + 1`` on and the first
    ``sinks`` of the sequence; pages in between are not read, and the table need not name them.
    That counts slots.  A tree's row lies in slot ``lengths[b] + t`` but at the position of its depth,
    where decoding its branch alone would put it: give ``positions``, int32 ``[batch, T]`` as
    ``kv8_append`` took them (between ``lengths[b]`` and ``lengths[b] + T - 1``, or the nearest of these),
    and the row sees of the context the slots from ``positions[b, t] - window + 1`` on, and of
    the block the rows that its bits name and whose positions are there (or below ``sinks``).
    ``counts`` int32 ``[batch]`` are the valid rows (None: T).  ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns ``(out, lse)``: ``out`` like ``q``, ``lse`` fp32 ``[batch, T,
    q_heads]``, the logarithm of each softmax's sum; rows that see nothing give 0 and -inf, rows
    that see a score of NaN or +inf NaN in both.

    Scores, maxima, sums and outputs are fp32.  A slot's weight meets its value as one f16 number
    for bf16 queries, as two for fp16 ones, which may put ``out``, before it is rounded, off by 2^-11 (2^-17) of
    the weighted sum of the values' magnitudes: more of what is left where values cancel.
    ``weight_parts=2`` has two parts for bf16 queries, too; blocks of many rows take longer.
    """
    _require_cache(cache, 8)
    if _elsewhere_current(cache):
        with torch.cuda.device(cache._index):
            return kv8_attention(q, cache, lengths, block=block, counts=counts, scale=scale, window=window,
                                 sinks=sinks, out=out, lse=lse, workspace=workspace, positions=positions,
                                 weight_parts=weight_parts)
    qp = _require_rows(q, cache, None, "q", _Q_DTYPES)
    batch, T, q_heads, D = q.shape
    if q_heads % cache.kv_heads:
        raise ValueError(f"{q_heads} query heads do not divide over {cache.kv_heads} key/value heads")
    if window is None:
        if sinks:
            raise ValueError("sinks are for a window")
        window = 0
    elif window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    else:
        window, sinks = min(window, _FAR), min(sinks, _FAR)
    lp, cp = _require_ints(lengths, cache, "lengths"), _require_ints(counts, cache, "counts")
    mode, mask, ld_mask = _block_args(block, cache, T)
    options = ()
    if positions is not None or weight_parts != 1:
        if weight_parts not in (1, 2):
            raise ValueError(f"weight_parts must be 1 or 2, got {weight_parts}")
        at = (None, 0)
        if positions is not None:
            if not window or mode != _lib.KV4_BLOCK_MASK:
                raise ValueError("positions are for a window over a block mask")
            at = _position_args(positions, cache, T)
        options = (ctypes.byref(_lib.Kv8OptionsParams(*at, weight_parts)),)
    if out is None:
        out = torch.empty(batch, T, q_heads, D, dtype=q.dtype, device=cache.device)
        op = (out.data_ptr(), T * q_heads * D, q_heads * D, D)
    else:
        op = _require_rows(out, cache, q_heads, "out", (q.dtype,))
        if out.shape != q.shape:
            raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    if lse is None:
        lse = torch.empty(batch, T, q_heads, dtype=torch.float32, device=cache.device)
    else:
        _require_lse(lse, cache, T, q_heads)
    lib = _lib.load()
    need = cache._ws_bytes.get((T, q_heads))
    if need is None:
        need = lib.dels_kv8_attention_ws_bytes(batch, T, q_heads, cache.kv_heads, D, cache.max_pages)
        cache._ws_bytes[T, q_heads] = need
    stream = _stream_ptr(cache.device)
    if workspace is None and not _capturing():
        ws = _WORKSPACES.get(cache.device, need, stream)
    else:
        ws = _own_workspace(workspace, cache, need, counters=True)
    call = lib.dels_kv8_attention_ex if options else lib.dels_kv8_attention
    _lib.check(call(cache._ref, *qp, _DTYPES[q.dtype], q_heads, T, lp, cp, mode, mask, ld_mask,
                    cache._scale if scale is None else scale, window, sinks, *options, *op, lse.data_ptr(),
                    ws.data_ptr(), ws.numel(), stream), call.__name__)
    return out, lse
