"""The paged key-value cache on B200: dense single-token attention over a pool of pages, and a
bounded cache that evicts by accumulated attention weight.

The reference bounds its window layers' cache by position and archives what leaves it
(pseudobrain/transplant.py:612-659, pseudobrain/exact_memory.py). This module is the other way
to keep a cache small, and the dense attention that a server needs beside both:

    PagedCache(k_pages, v_pages, mass, pos)     the pool (``PagedCache.allocate`` makes one)
    paged_append_(cache, k, v, ...)             new tokens into their sequences' pages
    paged_attend(cache, q, ...) -> (out, lse)   one new token per sequence over its cache, with
                                                an optional window and sinks; ``accumulate``
                                                adds the attention weights to the cache's mass
    paged_observe_(cache, q, ...)               the weights of a prompt's last queries into mass
    select_evictions(cache, ...)                which entries leave, as moves (src, dst, count)
    move_entries_(cache, ...)                   the moves
    paged_evict_(cache, ...)                    both: every sequence down to its budget

Keys and values are bf16 or fp16, [P, KV, page, hd] with hd 64, 128 or 256 and page a power of
two from 8 to 256 (any page, head and entry strides that are multiples of 8 elements). Entry i
of sequence b lies in page ``block_table[b, i // page]`` at row ``i % page``; ``block_table``
[B, M] and ``lengths`` [B] are int32 on the GPU and the caller's to keep: no call changes them,
none reads them on the host, so every call can be captured in a CUDA graph. A caller's step is

    paged_append_(cache, k, v, block_table, lengths, seen)
    lengths += 1; seen += 1
    out, lse = paged_attend(cache, q, block_table, lengths, accumulate=True)
    # every so often, when lengths may exceed the budget
    paged_evict_(cache, block_table, lengths, seen, budget, recent, sinks)
    lengths.clamp_(max=budget)

with the table, lengths and seen shared by all layers (each layer has a pool of its own). Grids,
move lists and workspaces follow the table's width, not the lengths on the device: once a prompt
is evicted, pass the columns that are left (``block_table[:, :pages]``, a view). With a table of
131072 entries instead, the choice for 64 x 8 heads of 4112 entries takes 222 us for 19, its moves
35 us for 3 and the attention of 8 x 4 heads with weights 36 us for 31. Rows
of a page past a sequence's length may hold anything; page ids outside the pool are never
followed. A page belongs to one sequence where a call writes it; attention without
``accumulate`` may read pages that several sequences share. Every kernel is CUDA (libpbk.so,
sm_100a); there is no CPU path, and no call has a backward pass: the attention refuses a query
that requires grad while gradients are recorded.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _capi
from ._capi import (LIB, PbkPagedAttendDesc, PbkPagedBatch, PbkPagedCache, PbkPagedObserveDesc, check)

_DTYPES = {torch.bfloat16: _capi.PBK_BF16, torch.float16: _capi.PBK_F16, torch.float32: _capi.PBK_F32}
_byref = ctypes.byref
_INT_MAX = 2 ** 31 - 1


def _same_places(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the elements of two tensors of one shape lie alike: the same strides, those of
    dimensions of one element aside (they may be anything)."""
    return a.stride() == b.stride() or all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


@dataclass
class PagedCache:
    """One layer's pool of pages: keys and values [P, KV, page, hd], and per entry and key head
    the accumulated attention weight ``mass`` (fp32) and the token's position ``pos`` (int32)
    [P, KV, page]. Calls that need a part say so when it is None. The tensors are not to be
    replaced once the cache is made (make another)."""
    k_pages: torch.Tensor | None
    v_pages: torch.Tensor | None
    mass: torch.Tensor | None = None
    pos: torch.Tensor | None = None

    def __post_init__(self):
        parts = [t for t in (self.k_pages, self.v_pages, self.mass, self.pos) if t is not None]
        if not parts:
            raise ValueError("paged cache: no tensors")
        self.device = parts[0].device
        if any(not t.is_cuda or t.device != self.device for t in parts):
            raise RuntimeError("paged cache: pseudobrain_b200 runs on CUDA only: every tensor must be on the same GPU "
                               "(there is no CPU fallback)")
        d = self._desc = PbkPagedCache()
        d.pages, d.kv, d.page = parts[0].shape[:3]
        if (self.k_pages is None) != (self.v_pages is None):
            raise ValueError("paged cache: keys and values come together")
        if self.k_pages is not None:
            k, v = self.k_pages, self.v_pages
            if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or not _same_places(k, v):
                raise ValueError("paged cache: k_pages and v_pages must be alike, [P, KV, page, hd]")
            if k.dtype not in (torch.bfloat16, torch.float16):
                raise TypeError(f"paged cache: bf16 or fp16 keys and values expected, got {k.dtype}")
            if k.stride(3) != 1:
                raise ValueError("paged cache: the last dim of k_pages and v_pages must be contiguous")
            d.d, d.dtype = k.shape[3], _DTYPES[k.dtype]
            d.k_pages, d.v_pages = k.data_ptr(), v.data_ptr()
            d.stride_page, d.stride_head, d.stride_entry = k.stride()[:3]
        meta = [t for t in (self.mass, self.pos) if t is not None]
        for t, name, dtype in ((self.mass, "mass", torch.float32), (self.pos, "pos", torch.int32)):
            if t is None:
                continue
            if t.shape != parts[0].shape[:3] or t.dtype != dtype or t.stride(2) != 1 or t.stride() != meta[0].stride():
                raise ValueError(f"paged cache: {name} must be {dtype} [P, KV, page] with contiguous entries, and mass "
                                 "and pos of the same strides")
            d.meta_page, d.meta_head = t.stride()[:2]
        d.mass = None if self.mass is None else self.mass.data_ptr()
        d.pos = None if self.pos is None else self.pos.data_ptr()
        self._ref, self._index, self._only_gpu = _byref(d), self.device.index, torch.cuda.device_count() == 1

    @classmethod
    def allocate(cls, pages: int, kv: int, page: int, hd: int, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda", weights: bool = True) -> "PagedCache":
        """A pool of ``pages`` pages (keys and values uninitialised); with ``weights`` also mass and
        pos, zeroed (for eviction)."""
        k = torch.empty(pages, kv, page, hd, dtype=dtype, device=device)
        mass = torch.zeros(pages, kv, page, dtype=torch.float32, device=device) if weights else None
        pos = torch.zeros(pages, kv, page, dtype=torch.int32, device=device) if weights else None
        return cls(k, torch.empty_like(k), mass, pos)

    @property
    def kv(self) -> int:
        return self._desc.kv

    @property
    def page(self) -> int:
        return self._desc.page


def _call(cache: PagedCache, fn, what: str, *args) -> None:
    """fn(*args, stream) on the cache's device and its current stream; raises on an error. A
    serving step makes many small calls, so the common case (that device is current) takes the
    stream's handle without making a Stream object."""
    i = cache._index
    if cache._only_gpu or torch.cuda.current_device() == i:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if status:
        check(status, what)


def _batch(cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor | None, seen: torch.Tensor | None = None):
    i = cache._index
    if table.dtype != torch.int32 or table.dim() != 2 or table.get_device() != i or (strides := table.stride())[1] != 1:
        raise ValueError("block_table must be int32 [B, M] on the cache's GPU with contiguous rows")
    b, m = table.shape
    return PbkPagedBatch(b, m, table.data_ptr(), strides[0],
                         None if lengths is None else _per_sequence(lengths, "lengths", b, i),
                         None if seen is None else _per_sequence(seen, "seen", b, i))


def _per_sequence(t: torch.Tensor, name: str, b: int, index: int) -> int:
    if t.dtype != torch.int32 or t.shape != (b,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{b}] on the cache's GPU")
    return t.data_ptr()


def _need(cache: PagedCache, what: str, *names: str) -> None:
    for n in names:
        if getattr(cache, n) is None:
            raise ValueError(f"{what}: the cache has no {n}")


def _rows(t: torch.Tensor, cache: PagedCache, what: str) -> None:
    k = cache.k_pages
    if t.get_device() != cache._index or t.dtype != k.dtype or t.size(-1) != cache._desc.d or t.stride(-1) != 1:
        raise ValueError(f"{what}: {k.dtype} with a contiguous last dim of {k.shape[3]} on the cache's GPU expected, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _run(cache: PagedCache, fn, workspace, what: str, *args) -> None:
    """_call with a workspace of workspace(*args) bytes from the caching allocator behind the other
    arguments. Its size follows the current device's SMs and the clusters that it holds, so it is
    asked for where the call will run."""
    if not cache._only_gpu and torch.cuda.current_device() != cache._index:
        with torch.cuda.device(cache._index):
            return _run(cache, fn, workspace, what, *args)
    nbytes = workspace(*args)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=cache.device)
        _call(cache, fn, what, *args, ws.data_ptr(), nbytes)
    else:
        _call(cache, fn, what, *args, None, 0)


def paged_append_(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                  lengths: torch.Tensor, seen: torch.Tensor | None = None,
                  cu_seqlens: torch.Tensor | None = None) -> None:
    """Put new tokens into the cache: k, v [N, KV, hd] of the same strides; sequence b's are rows
    cu_seqlens[b] .. cu_seqlens[b+1] - 1 (int32 [B+1]; None: one token per sequence, N == B). Its
    i-th becomes entry lengths[b] + i, with mass 0 and position seen[b] + i (lengths[b] + i without ``seen``).
    Tokens past the table's capacity are left out."""
    _need(cache, "paged_append_", "k_pages")
    _rows(k, cache, "k")
    shape, strides = k.shape, k.stride()
    if len(shape) != 3 or shape[1] != cache._desc.kv or v.shape != shape or v.dtype != k.dtype \
            or not _same_places(k, v) or v.get_device() != cache._index:
        raise ValueError(f"paged_append_: k and v must be alike, [N, {cache.kv}, hd] with the same strides, got "
                         f"{tuple(k.shape)} {strides} and {tuple(v.shape)} {v.stride()}")
    b = _batch(cache, block_table, lengths, seen)
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.shape != (b.batch + 1,) or not cu_seqlens.is_contiguous() \
                or cu_seqlens.device != cache.device:
            raise ValueError(f"cu_seqlens must be contiguous int32 [{b.batch + 1}] on the cache's GPU")
    elif shape[0] != b.batch:
        raise ValueError(f"paged_append_: {shape[0]} tokens for {b.batch} sequences need cu_seqlens")
    _call(cache, LIB.pbk_paged_append, "pbk_paged_append", cache._ref, _byref(b), k.data_ptr(), v.data_ptr(),
          strides[0], strides[1], shape[0], None if cu_seqlens is None else cu_seqlens.data_ptr())


def paged_attend(cache: PagedCache, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                 window: int | None = None, sinks: int = 0, scale: float | None = None, accumulate: bool = False,
                 out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of one new token per sequence: q [B, H, hd] over the lengths[b] entries of each
    sequence (the token's own among them), of which the first ``sinks`` and the last ``window``
    are visible (all when window is None; entries count, so a window is for a cache whose
    entries lie in order). Returns out [B, H, hd] in q's dtype (or ``out``, which may be fp32)
    and lse [B, H], the natural logarithm of the sum of exponentials. Scores and sums are fp32;
    weights meet the values with 16 bits (bf16 caches) or 22 (fp16 caches), so an fp32 ``out``
    holds about 5 or 6 digits. A sequence without entries gives 0 and -inf. ``accumulate`` adds
    every entry's weight, summed over the query heads of its key head, to cache.mass; it takes a
    workspace of 4 bytes per query head and entry that the table (or the window and sinks) has
    room for."""
    _need(cache, "paged_attend", "k_pages")
    if torch.is_grad_enabled() and (q.requires_grad or cache.k_pages.requires_grad or cache.v_pages.requires_grad):
        raise RuntimeError("paged_attend has no backward pass: call it under torch.no_grad() or on detached tensors")
    if accumulate:
        _need(cache, "paged_attend", "mass")
    _rows(q, cache, "q")
    b = _batch(cache, block_table, lengths)
    if q.dim() != 3 or (shape := q.shape)[0] != b.batch:
        raise ValueError(f"paged_attend: q must be [{b.batch}, H, hd], got {tuple(q.shape)}")
    if window is not None and window < 1:
        raise ValueError("paged_attend: the window holds at least the new token (None: no window)")
    n, h, d = shape
    sb, sh, _ = q.stride()
    if out is None:
        out, ob, oh, dtype = torch.empty_like(q, memory_format=torch.contiguous_format), h * d, d, cache._desc.dtype
    elif out.shape != shape or out.dtype not in (q.dtype, torch.float32) or out.stride(-1) != 1 \
            or out.device != q.device:
        raise ValueError(f"paged_attend: out must be {tuple(shape)}, {q.dtype} or fp32, with a contiguous last dim")
    else:
        (ob, oh, _), dtype = out.stride(), _DTYPES[out.dtype]
    lse = torch.empty(n, h, dtype=torch.float32, device=cache.device)
    desc = PbkPagedAttendDesc(h, 0 if window is None else min(window, _INT_MAX), min(sinks, _INT_MAX), accumulate,
                              d ** -0.5 if scale is None else scale, dtype, q.data_ptr(), sb, sh, out.data_ptr(), ob, oh,
                              lse.data_ptr())
    _run(cache, LIB.pbk_paged_attend, LIB.pbk_paged_attend_workspace, "pbk_paged_attend", cache._ref, _byref(b), _byref(desc))
    return out, lse


def paged_observe_(cache: PagedCache, q: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                   scale: float | None = None) -> None:
    """Add to cache.mass the attention weights of each sequence's last W tokens, q [B, W, H, hd]
    (their queries; the tokens are the sequence's last W entries, and each sees the entries up
    to its own), summed over them and over the query heads of the key head. Of a sequence
    shorter than W the last lengths[b] queries count. After a prompt this tells the eviction
    what the prompt's end attends to."""
    _need(cache, "paged_observe_", "k_pages", "mass")
    _rows(q, cache, "q")
    b = _batch(cache, block_table, lengths)
    if q.dim() != 4 or q.shape[0] != b.batch:
        raise ValueError(f"paged_observe_: q must be [{b.batch}, W, H, hd], got {tuple(q.shape)}")
    desc = PbkPagedObserveDesc(q.shape[2], q.shape[1], q.shape[3] ** -0.5 if scale is None else scale, 0, q.data_ptr(),
                               q.stride(0), q.stride(1), q.stride(2))
    _run(cache, LIB.pbk_paged_observe, LIB.pbk_paged_observe_workspace, "pbk_paged_observe", cache._ref, _byref(b),
         _byref(desc))


def select_evictions(cache: PagedCache, block_table: torch.Tensor, lengths: torch.Tensor, seen: torch.Tensor,
                     budget: int, recent: int = 0, sinks: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Choose, for each sequence with more than ``budget`` entries and each key head, the
    ``budget`` entries that stay: those at positions below ``sinks`` and the last ``recent`` of
    the ``seen`` positions first, then by mass downwards (NaN above every number, ties to the
    lowest entry). Returns the moves that bring them below ``budget``: src and dst int32
    [B, KV, moves] (ascending; -1 past the count; moves = min(budget, M * page - budget)) and
    count int32 [B, KV]. Nothing is moved."""
    _need(cache, "select_evictions", "mass", "pos")
    b = _batch(cache, block_table, lengths, seen)
    if budget < 1 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("select_evictions: budget >= 1 and recent + sinks <= budget expected")
    moves = max(0, min(budget, b.width * cache.page - budget))
    places = torch.empty(2, b.batch, cache.kv, moves, dtype=torch.int32, device=cache.device)
    src, dst = places.unbind(0)
    count = torch.empty(b.batch, cache.kv, dtype=torch.int32, device=cache.device)
    _call(cache, LIB.pbk_paged_select, "pbk_paged_select", cache._ref, _byref(b), budget, recent, sinks, src.data_ptr(),
          dst.data_ptr(), count.data_ptr(), moves)
    return src, dst, count


def move_entries_(cache: PagedCache, block_table: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
                  count: torch.Tensor) -> None:
    """Entry dst[b, h, n] := entry src[b, h, n] for n < count[b, h]: key, value, and mass and pos
    where the cache has them. No place in dst may be a source."""
    _need(cache, "move_entries_", "k_pages")
    b = _batch(cache, block_table, None)
    if src.dim() != 3 or src.shape[:2] != (b.batch, cache.kv) or dst.shape != src.shape or count.shape != src.shape[:2]:
        raise ValueError(f"move_entries_: src and dst must be [{b.batch}, {cache.kv}, n] and count their first two dims")
    for t, name in ((src, "src"), (dst, "dst"), (count, "count")):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != cache.device:
            raise ValueError(f"move_entries_: {name} must be contiguous int32 on the cache's GPU")
    _call(cache, LIB.pbk_paged_move, "pbk_paged_move", cache._ref, _byref(b), src.data_ptr(), dst.data_ptr(),
          count.data_ptr(), src.size(2))


def paged_evict_(cache: PagedCache, block_table: torch.Tensor, lengths: torch.Tensor, seen: torch.Tensor, budget: int,
                 recent: int = 0, sinks: int = 0) -> None:
    """Bring every sequence down to ``budget`` entries (select_evictions, then move_entries_).
    Afterwards a sequence that had more has its entries at 0 .. budget - 1, in no particular
    order: the caller's lengths become min(lengths, budget)."""
    _need(cache, "paged_evict_", "k_pages")
    src, dst, count = select_evictions(cache, block_table, lengths, seen, budget, recent, sinks)
    move_entries_(cache, block_table, src, dst, count)
