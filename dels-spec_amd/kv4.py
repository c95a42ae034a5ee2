"""Key/value cache held in 4 bits, and attention over it (gfx950 kernels).

The target's side of a draft block's verification (code/dflash.py:637-651): the
block's keys and values enter the cache, its queries attend over context and
block, rejected rows are cropped by going on from a shorter length.  The
reference keeps the cache in bf16 inside transformers; here it is pages of 64
slots in 4 bits a value (include/dels.h describes a page), which a sequence's row
of page numbers names.  Lengths live on the GPU and no call reads them back, so
every call can be captured into a graph.  A captured call has a workspace of its
own, from the graph's memory, whose counters a node of the graph clears; one that is
given (``workspace``, from ``ops.new_workspace``) saves that node and is the caller's to
keep: calls that share it must not overlap, in whatever graphs and streams they are.

  * ``kv4_append``    -- a block's rows into the cache
  * ``kv4_read``      -- the values that slots of the cache stand for
  * ``kv4_attention`` -- attention of a block's rows, one token or a prompt's chunk
  * ``kv4_weights``   -- the attention weights that accepted rows gave to each slot
  * ``kv4_evict``     -- drop the slots of least weight

A length is the number of slots a sequence holds *before* the block, in all calls
alike: row ``t`` of a block lies in slot ``lengths[b] + t``.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib
from .ops import _DTYPES, _WORKSPACES, _require_cuda, _stream_ptr

PAGE = 64              # slots of a page
HEAD_DIMS = (64, 128)
_CONTROL_BYTES = 1 << 16    # a workspace's control area (include/dels.h): the arrival counters lie there


def page_bytes(head_dim: int) -> int:
    """Bytes of one key/value head's page of 64 slots."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    return 66 * head_dim + 128


def _row_stride(t: torch.Tensor, columns: int, name: str) -> int:
    """Row stride of a 2-d tensor: 0 where all rows are one (an expanded tensor), else at least ``columns``."""
    stride = t.stride(0)
    if t.shape[0] <= 1:
        return columns                     # one row: no stride that matters
    if 0 < stride < columns:
        raise ValueError(f"{name} must not have overlapping rows (row stride {stride}, {columns} columns)")
    return stride


class PagedCache:
    """Pages of a key/value cache and the table that hands them out; a class a format.

    ``data`` uint8 ``[num_pages, kv_heads, page_bytes(head_dim)]``, contiguous;
    ``block_table`` int32 ``[batch, max_pages]``, unit column stride: slot ``j`` of
    sequence ``b`` is slot ``j % 64`` of page ``block_table[b, j // 64]``.  Entries
    outside ``[0, num_pages)`` name no page.  Pages may be shared by sequences that
    only read them, and a whole row by an expanded table.  The cache keeps both
    tensors; a table can be rewritten in place.
    """

    bits: int              # of a key or value

    @staticmethod
    def page_bytes(head_dim: int) -> int:
        """Bytes of one key/value head's page of 64 slots."""
        raise NotImplementedError

    def __init__(self, data: torch.Tensor, block_table: torch.Tensor, head_dim: int):
        _require_cuda(data, "data")
        _require_cuda(block_table, "block_table")
        if data.dtype != torch.uint8 or data.dim() != 3 or data.shape[2] != self.page_bytes(head_dim):
            raise ValueError(f"data must be uint8 [num_pages, kv_heads, {self.page_bytes(head_dim)}], got "
                             f"{data.dtype} {tuple(data.shape)}")
        if data.shape[1] < 1:
            raise ValueError("data must have one key/value head at least")
        if not data.is_contiguous():
            raise ValueError("data must be contiguous")
        if block_table.dtype != torch.int32 or block_table.dim() != 2:
            raise ValueError("block_table must be int32 [batch, max_pages]")
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table must have unit column stride")
        if block_table.device != data.device:
            raise ValueError("data and block_table must be on one device")
        self.data = data
        self.block_table = block_table
        self.head_dim = int(head_dim)
        self.kv_heads = int(data.shape[1])
        self.batch, self.max_pages = (int(x) for x in block_table.shape)
        self.slots = self.max_pages * PAGE
        self.device = data.device
        self._index = data.get_device()
        self._scale = self.head_dim ** -0.5
        self._ws_bytes = {}                    # attention's workspace size by (T, q_heads)
        self._params = _lib.Kv4CacheParams(data.data_ptr(), data.shape[0], self.kv_heads, self.head_dim,
                                           block_table.data_ptr(),
                                           _row_stride(block_table, self.max_pages, "block_table"),
                                           self.batch, self.max_pages)
        self._ref = ctypes.byref(self._params)

    @classmethod
    def allocate(cls, batch: int, max_len: int, kv_heads: int, head_dim: int, device) -> "PagedCache":
        """An empty cache in which every sequence owns the pages of ``max_len`` slots."""
        pages = -(-max_len // PAGE)
        data = torch.zeros(batch * pages, kv_heads, cls.page_bytes(head_dim), dtype=torch.uint8, device=device)
        table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        return cls(data, table, head_dim)


class KV4Cache(PagedCache):
    """Pages of a 4-bit key/value cache and the table that hands them out (``PagedCache`` says how)."""

    bits = 4
    page_bytes = staticmethod(page_bytes)


def _require_cache(cache: PagedCache, bits: int) -> None:
    """Refuse a cache of the other format: its pages have another size."""
    if cache.bits != bits:
        raise TypeError(f"cache holds {cache.bits} bits a value, the call is for {bits}")


def _elsewhere(t, cache: PagedCache, name: str) -> None:
    """Raise for a tensor that is not on the cache's GPU."""
    _require_cuda(t, name)
    raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")


def _require_ints(t: Optional[torch.Tensor], cache: PagedCache, name: str) -> Optional[int]:
    """Pointer of an int32 [batch] device array (None where there is none)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.get_device() != cache._index:
        _elsewhere(t, cache, name)
    if t.dtype != torch.int32 or t.shape != (cache.batch,):
        raise ValueError(f"{name} must be int32 [{cache.batch}], got {t.dtype} {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _require_rows(t: torch.Tensor, cache: PagedCache, heads: Optional[int], name: str,
                  dtypes) -> tuple[int, int, int, int]:
    """(pointer, strides) of a [batch, T, heads, head_dim] tensor with unit channel stride."""
    if not isinstance(t, torch.Tensor) or t.get_device() != cache._index:
        _elsewhere(t, cache, name)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} dtype {t.dtype} not supported")
    shape = t.shape
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != cache.head_dim or (
            heads is not None and shape[2] != heads):
        raise ValueError(f"{name} must be [{cache.batch}, T, {'heads' if heads is None else heads}, "
                         f"{cache.head_dim}], got {tuple(shape)}")
    sb, st, sh, sc = t.stride()
    if sc != 1:
        raise ValueError(f"{name} must have unit channel stride")
    # a dimension of one has no stride that matters
    return (t.data_ptr(), sb if shape[0] > 1 else 0, st if shape[1] > 1 else 0, sh if shape[2] > 1 else 0)


# whether the current stream is being captured, without the wrapper's call
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _own_workspace(given: Optional[torch.Tensor], cache: PagedCache, need: int, *, counters: bool) -> torch.Tensor:
    """The caller's workspace, or else a captured call's own.

    The stream's shared one may be replaced by a larger one between a graph's replays, its
    zero fill would belong to the one graph that captured it, and graphs that are replayed
    on several streams would meet in it.
    """
    if given is not None:
        if not isinstance(given, torch.Tensor) or given.get_device() != cache._index:
            _elsewhere(given, cache, "workspace")
        if given.dtype != torch.uint8 or not given.is_contiguous():
            raise ValueError("workspace must be contiguous uint8")
        return given
    ws = torch.empty(need, dtype=torch.uint8, device=cache.device)
    if counters:
        ws[:_CONTROL_BYTES].zero_()
    return ws


_Q_DTYPES = (torch.bfloat16, torch.float16)


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, *,
               counts: Optional[torch.Tensor] = None) -> None:
    """Write rows ``t < counts[b]`` (None: all) of ``k`` and ``v`` into slots ``lengths[b] + t``.

    ``k``, ``v`` ``[batch, T, kv_heads, head_dim]`` fp32, bf16 or fp16, any strides that
    keep rows 16-byte aligned.  ``lengths`` is not changed; rows past the table's
    slots are dropped.
    """
    _require_cache(cache, 4)
    kp = _require_rows(k, cache, cache.kv_heads, "k", _DTYPES)
    vp = _require_rows(v, cache, cache.kv_heads, "v", _DTYPES)
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError("k and v must have one shape and dtype")
    lp, cp = _require_ints(lengths, cache, "lengths"), _require_ints(counts, cache, "counts")
    lib = _lib.load()
    _lib.check(lib.dels_kv4_append(cache._ref, *kp, *vp, _DTYPES[k.dtype], lp, cp, k.shape[1],
                                   _stream_ptr(cache.device)), "dels_kv4_append")


def kv4_read(cache: KV4Cache, starts: torch.Tensor, T: int, *, counts: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that slots ``starts[b] + t``, ``t < T``, stand for.

    Returns ``(k, v)``, each ``[batch, T, kv_heads, head_dim]`` of ``dtype``; zeros from
    ``counts[b]`` on (None: none) and past the table's slots.
    """
    _require_cache(cache, 4)
    if dtype not in _DTYPES:
        raise TypeError(f"dtype {dtype} not supported")
    sp, cp = _require_ints(starts, cache, "starts"), _require_ints(counts, cache, "counts")
    k = torch.empty(cache.batch, T, cache.kv_heads, cache.head_dim, dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    lib = _lib.load()
    _lib.check(lib.dels_kv4_read(cache._ref, sp, cp, T, k.data_ptr(), v.data_ptr(), _DTYPES[dtype],
                                 _stream_ptr(cache.device)), "dels_kv4_read")
    return k, v


Block = Union[str, torch.Tensor]


def _block_args(block: Block, cache: PagedCache, T: int) -> tuple[int, Optional[int], int]:
    """(mode, mask pointer, mask row stride)."""
    if isinstance(block, torch.Tensor):
        if block.get_device() != cache._index:
            _elsewhere(block, cache, "block")
        if block.dtype != torch.int64 or block.shape != (cache.batch, T):
            raise ValueError(f"a block mask must be int64 [{cache.batch}, {T}], got {block.dtype} "
                             f"{tuple(block.shape)}")
        if T > 1 and block.stride(1) != 1:
            raise ValueError("a block mask must have unit column stride")
        return _lib.KV4_BLOCK_MASK, block.data_ptr(), _row_stride(block, T, "a block mask")
    if block not in _lib.KV4_BLOCK_CODES:
        raise ValueError(f"block must be one of {sorted(_lib.KV4_BLOCK_CODES)} or an int64 mask, got {block!r}")
    return _lib.KV4_BLOCK_CODES[block], None, 0


def kv4_attention(q: torch.Tensor, cache: KV4Cache, lengths: torch.Tensor, *, block: Block = "causal",
                  counts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of a block's rows over their sequences' context and the block itself.

    ``q`` ``[batch, T, q_heads, head_dim]`` bf16 or fp16, ``q_heads`` a multiple of the
    cache's heads (fp16 needs keys below 2^20 in magnitude, and takes them as multiples of
    2^-20).  Every row sees slots ``[0, lengths[b])``; of the block's own slots
    (which ``kv4_append`` wrote) ``block`` says which: ``"causal"``, ``"full"``, ``"none"``, or
    an int64 ``[batch, T]`` of bits, bit ``i`` of row ``t`` for slot ``lengths[b] + i`` (a tree of
    drafts; T at most 64; expanded where all sequences have one tree).  ``counts`` int32
    ``[batch]`` are the valid rows (None: T).  ``scale`` defaults to ``head_dim ** -0.5``.
    Returns ``(out, lse)``: ``out`` like ``q``, ``lse`` fp32 ``[batch, T, q_heads]``, the
    logarithm of each softmax's sum; rows that see nothing give 0 and -inf, rows that see
    a score of NaN or +inf NaN in both.
    """
    _require_cache(cache, 4)
    qp = _require_rows(q, cache, None, "q", _Q_DTYPES)
    batch, T, q_heads, D = q.shape
    if q_heads % cache.kv_heads:
        raise ValueError(f"{q_heads} query heads do not divide over {cache.kv_heads} key/value heads")
    lp, cp = _require_ints(lengths, cache, "lengths"), _require_ints(counts, cache, "counts")
    mode, mask, ld_mask = _block_args(block, cache, T)
    if out is None:
        out = torch.empty(batch, T, q_heads, D, dtype=q.dtype, device=cache.device)
        s = T * q_heads * D, q_heads * D, D
        op = (out.data_ptr(), *s)
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
        need = lib.dels_kv4_attention_ws_bytes(batch, T, q_heads, cache.kv_heads, D, cache.max_pages)
        cache._ws_bytes[T, q_heads] = need
    stream = _stream_ptr(cache.device)
    if workspace is None and not _capturing():
        ws = _WORKSPACES.get(cache.device, need, stream)
    else:
        ws = _own_workspace(workspace, cache, need, counters=True)
    _lib.check(lib.dels_kv4_attention(cache._ref, *qp, _DTYPES[q.dtype], q_heads, T, lp, cp, mode, mask, ld_mask,
                                      cache._scale if scale is None else scale, *op, lse.data_ptr(),
                                      ws.data_ptr(), ws.numel(), stream), "dels_kv4_attention")
    return out, lse


def _require_lse(lse: torch.Tensor, cache: PagedCache, T: int, q_heads: int) -> None:
    if not isinstance(lse, torch.Tensor) or lse.get_device() != cache._index:
        _elsewhere(lse, cache, "lse")
    if lse.dtype != torch.float32 or lse.shape != (cache.batch, T, q_heads) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous float32 [{cache.batch}, {T}, {q_heads}], got {lse.dtype} "
                         f"{tuple(lse.shape)}")


def _require_weights(w: torch.Tensor, cache: KV4Cache, name: str) -> None:
    if not isinstance(w, torch.Tensor) or w.get_device() != cache._index:
        _elsewhere(w, cache, name)
    if w.dtype != torch.float32 or w.shape != (cache.batch, cache.kv_heads, cache.slots) or not w.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 [{cache.batch}, {cache.kv_heads}, {cache.slots}], got "
                         f"{w.dtype} {tuple(w.shape)}")


def kv4_weights(q: torch.Tensor, cache: KV4Cache, lengths: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor,
                accepted: Optional[torch.Tensor] = None, *, block: Block = "causal",
                counts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Add the attention weights that the rows ``t < accepted[b]`` gave to each slot.

    The other arguments as ``kv4_attention`` had them, ``lse`` as it returned it.
    ``weights`` fp32 ``[batch, kv_heads, cache.slots]``: the result is, for slots of the
    context, ``weights`` plus the softmax weights of the accepted rows (None: all
    valid rows) summed over the query heads of each cache head; the block's own slots
    start from 0, and slots past the block are 0.  ``out`` may be ``weights``.
    """
    _require_cache(cache, 4)
    qp = _require_rows(q, cache, None, "q", _Q_DTYPES)
    batch, T, q_heads, D = q.shape
    if q_heads % cache.kv_heads:
        raise ValueError(f"{q_heads} query heads do not divide over {cache.kv_heads} key/value heads")
    lp, cp = _require_ints(lengths, cache, "lengths"), _require_ints(counts, cache, "counts")
    ap = _require_ints(accepted, cache, "accepted")
    mode, mask, ld_mask = _block_args(block, cache, T)
    if not isinstance(lse, torch.Tensor) or lse.get_device() != cache._index:
        _elsewhere(lse, cache, "lse")
    if lse.dtype == torch.float32 and not lse.is_contiguous():
        lse = lse.contiguous()
    _require_lse(lse, cache, T, q_heads)
    _require_weights(weights, cache, "weights")
    if out is None:
        out = torch.empty_like(weights)
    else:
        _require_weights(out, cache, "out")
    lib = _lib.load()
    _lib.check(lib.dels_kv4_weights(cache._ref, *qp, _DTYPES[q.dtype], q_heads, T, lp, cp, ap, mode, mask, ld_mask,
                                    cache._scale if scale is None else scale, lse.data_ptr(),
                                    weights.data_ptr(), out.data_ptr(), _stream_ptr(cache.device)),
               "dels_kv4_weights")
    return out


def kv4_evict(cache: KV4Cache, lengths: torch.Tensor, weights: torch.Tensor, keep: int, recent: int = 0, *,
              workspace: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Shrink every sequence of more than ``keep`` slots to ``keep``, each cache head by its own weights.

    The last ``recent`` slots (at most ``keep``) stay, and of the others those of
    largest weight (equal weights: lowest slot; NaN as -inf).  Slots that stay from
    ``keep`` on move into the places given up below it, both in ascending order; the
    cache changes in place.  Returns ``(lengths, weights, source)``: the new lengths, the
    weights in their new places (0 past them), and int32 ``source`` ``[batch, kv_heads,
    keep]``, the slot whose content each place holds now (-1 past the new length), by
    which whatever else is kept per slot follows.  Slots of a table entry that names no
    page hold nothing, so none of them stays or moves, and as places they take nothing.
    """
    _require_cache(cache, 4)
    lp = _require_ints(lengths, cache, "lengths")
    _require_weights(weights, cache, "weights")
    if keep < 1 or recent < 0:
        raise ValueError(f"keep must be at least 1 and recent at least 0, got {keep} and {recent}")
    new_lengths = torch.empty_like(lengths)
    new_weights = torch.empty_like(weights)
    source = torch.empty(cache.batch, cache.kv_heads, keep, dtype=torch.int32, device=cache.device)
    lib = _lib.load()
    need = lib.dels_kv4_evict_ws_bytes(cache.batch, cache.kv_heads, keep)
    stream = _stream_ptr(cache.device)
    if workspace is None and not _capturing():
        ws = _WORKSPACES.get(cache.device, need, stream)
    else:
        ws = _own_workspace(workspace, cache, need, counters=False)
    _lib.check(lib.dels_kv4_evict(cache._ref, lp, weights.data_ptr(), keep, recent, new_lengths.data_ptr(),
                                  new_weights.data_ptr(), source.data_ptr(), ws.data_ptr(), ws.numel(), stream),
               "dels_kv4_evict")
    return new_lengths, new_weights, source
