"""A paged key/value cache in device memory and attention over it, on resident handles.

The reference names the object (the ``cache`` and ``kv_state`` parameters of ``flash_attn``,
``python/tessera/__init__.py:1304-1317``) and has no device form of it.  Three calls make up a step of a program that
serves a model, all enqueued on the default stream:

    cache = PagedKVCache(num_pages=4096, page_size=16, num_kv_heads=8, head_dim=128, quant="e4m3")
    pages = SequencePages(cache)
    step = pages.extend({seq: new_tokens, ...})      # pages for the new tokens; slots, tables and lengths on the device
    cache.write(k, v, step.slots)                    # K and V of the new tokens, [T, Hkv, D]
    o = paged_attention(q, cache, step)              # [T, Hq, D]: single tokens and chunks in one batch

or, from one fused projection, ``write_fused_qkv`` and ``paged_attention_fused_qkv`` (``examples/paged_serving.py``).

:class:`SequencePages` is host bookkeeping and optional: a program with its own allocator passes a :class:`PagedBatch`
of its own arrays.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Dict, Hashable, List, Optional

import numpy as np

from . import lane as _lane
from .resident import DeviceArray, _result

_FORMAT = {None: 0, "i8": 1, "e4m3": 2}
_CODES = {"i8": "i8", "e4m3": "u8"}


class PagedKVCache:
    """K and V of ``num_pages`` pages of ``page_size`` slots, ``num_kv_heads`` heads of ``head_dim``.

    ``dtype``: the 16-bit type of the program, ``"bf16"`` or ``"f16"``.  ``quant``: ``None`` keeps it in the cache,
    ``"i8"`` and ``"e4m3"`` keep 8-bit codes with one f32 scale for each slot and head.  ``layout``: ``"nhd"`` is
    [pages, page_size, heads, D] in memory, ``"hnd"`` [pages, heads, page_size, D].  Cleared when it is made."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *, dtype: str = "bf16",
                 quant: Optional[str] = None, layout: str = "nhd"):
        if dtype not in ("bf16", "f16"):
            raise ValueError("dtype must be 'bf16' or 'f16'")
        if quant not in _FORMAT:
            raise ValueError("quant must be None, 'i8' or 'e4m3'")
        if layout not in ("nhd", "hnd"):
            raise ValueError("layout must be 'nhd' or 'hnd'")
        if min(num_pages, page_size, num_kv_heads, head_dim) <= 0 or head_dim % 16 or head_dim > 256:
            raise ValueError("sizes must be positive, head_dim a multiple of 16 and at most 256")
        if num_pages * page_size > 0x7fffffff:
            raise ValueError("a cache has at most 2**31 - 1 slots")
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = num_pages, page_size, num_kv_heads, head_dim
        self.dtype, self.quant, self.layout = dtype, quant, layout
        nhd = layout == "nhd"
        outer = (num_pages, page_size, num_kv_heads) if nhd else (num_pages, num_kv_heads, page_size)
        tag = dtype if quant is None else _CODES[quant]

        def cleared(shape, tag):
            a = DeviceArray(shape, tag, _lane.DeviceBuffer(math.prod(shape) * {"bf16": 2, "f16": 2, "f32": 4}.get(tag, 1)))
            a.buf.zero()
            return a

        self.k, self.v = cleared(outer + (head_dim,), tag), cleared(outer + (head_dim,), tag)
        self.k_scale = self.v_scale = None
        if quant is not None:
            self.k_scale, self.v_scale = cleared(outer, "f32"), cleared(outer, "f32")

        def strides(width):
            page, inner, innermost = page_size * num_kv_heads * width, outer[2] * width, width
            return (page, inner, innermost) if nhd else (page, innermost, inner)

        self.handle = _lane.KVCache(
            k=self.k.ptr, v=self.v.ptr, k_scale=self.k_scale.ptr if quant else None, v_scale=self.v_scale.ptr if quant else None,
            k_strides=strides(head_dim), v_strides=strides(head_dim), scale_strides=strides(1), num_pages=num_pages,
            page_size=page_size, num_heads=num_kv_heads, head_dim=head_dim, format=_FORMAT[quant])

    @property
    def num_slots(self) -> int:
        return self.num_pages * self.page_size

    def _rows(self, x: DeviceArray, name: str) -> DeviceArray:
        if x.dtype != self.dtype or x.ndim != 3 or x.shape[1:] != (self.num_kv_heads, self.head_dim):
            raise ValueError(f"{name} must be {self.dtype} (T, {self.num_kv_heads}, {self.head_dim}); got {x.dtype} {x.shape}")
        return x

    def _strides(self):
        row = self.num_kv_heads * self.head_dim
        return (ctypes.c_int64 * 4)(row, self.head_dim, row, self.head_dim)

    def _slots(self, slots: DeviceArray, tokens: Optional[int] = None) -> int:
        if slots.dtype != "i64" or slots.ndim != 1 or (tokens is not None and slots.shape[0] != tokens):
            raise ValueError(f"slots must be i64 ({'T' if tokens is None else tokens},); got {slots.dtype} {slots.shape}")
        return slots.shape[0]

    def write(self, K: DeviceArray, V: DeviceArray, slots: DeviceArray) -> None:
        """Token ``t``'s rows ``K[t]``, ``V[t]`` go to slot ``slots[t]`` (quantised on the way); a slot outside of the
        cache leaves its token out, two tokens of one call may not share one."""
        K, V = self._rows(K, "K"), self._rows(V, "V")
        T = self._slots(slots, K.shape[0])
        if V.shape != K.shape:
            raise ValueError(f"K {K.shape} and V {V.shape} differ")
        fn = getattr(_lane.load(), f"tessera_gfx950_kv_cache_write_{self.dtype}_dev")
        _lane.check(fn(ctypes.byref(self.handle), K.address, V.address, self._strides(), slots.address, T, None), "kv_cache_write")

    def write_fused_qkv(self, QKV: DeviceArray, num_q_heads: int, slots: DeviceArray) -> None:
        """The same from the output of one fused projection, ``QKV [T, (Hq + 2 Hkv) * D]``: the K and V column
        blocks are read where they lie."""
        width = (num_q_heads + 2 * self.num_kv_heads) * self.head_dim
        if QKV.dtype != self.dtype or QKV.ndim != 2 or QKV.shape[1] != width:
            raise ValueError(f"QKV must be {self.dtype} (T, {width}); got {QKV.dtype} {QKV.shape}")
        T = self._slots(slots, QKV.shape[0])
        k = QKV.address + num_q_heads * self.head_dim * 2
        fn = getattr(_lane.load(), f"tessera_gfx950_kv_cache_write_{self.dtype}_dev")
        strides = (ctypes.c_int64 * 4)(width, self.head_dim, width, self.head_dim)
        _lane.check(fn(ctypes.byref(self.handle), k, k + self.num_kv_heads * self.head_dim * 2, strides, slots.address, T, None),
                    "kv_cache_write")

    def read(self, slots: DeviceArray):
        """``K, V [T, Hkv, D]`` of the slots in the 16-bit type (zeros for a slot outside of the cache)."""
        T = self._slots(slots)
        shape = (T, self.num_kv_heads, self.head_dim)
        K, V = _result(shape, self.dtype), _result(shape, self.dtype)
        fn = getattr(_lane.load(), f"tessera_gfx950_kv_cache_read_{self.dtype}_dev")
        _lane.check(fn(ctypes.byref(self.handle), slots.address, K.address, V.address, self._strides(), T, None), "kv_cache_read")
        return K, V


@dataclass
class PagedBatch:
    """One call's sequences: their new tokens are rows ``q_offsets[b] .. q_offsets[b + 1]`` of Q, their keys (the new ones
    among them) ``kv_lens[b]`` slots through ``page_table[b]``; ``slots`` are the new tokens' own.  A Q has as many rows as there
    are slots; a batch of fewer rows than were written (the last token of each sequence, say) leaves the slots out.  Rows that
    no sequence has (where slots outside of the cache fill a batch up) are not written."""
    slots: Optional[DeviceArray]    # i64 [T]
    page_table: DeviceArray     # i32 [B, pages]
    q_offsets: DeviceArray      # i32 [B + 1]
    kv_lens: DeviceArray        # i32 [B]
    max_q: int
    max_kv: int


class SequencePages:
    """Host bookkeeping of which sequence holds which pages of a cache."""

    def __init__(self, cache: PagedKVCache):
        self.cache = cache
        self._free: List[int] = list(range(cache.num_pages - 1, -1, -1))
        self._pages: Dict[Hashable, List[int]] = {}
        self._length: Dict[Hashable, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: Hashable) -> int:
        return self._length.get(seq, 0)

    def slots(self, seq: Hashable, first: int = 0, last: Optional[int] = None) -> np.ndarray:
        """Slot numbers of a sequence's tokens [first, last), as ``read`` takes them; ``IndexError`` past its end."""
        end = self.length(seq)
        last = end if last is None else last
        if not 0 <= first <= last <= end:
            raise IndexError(f"tokens [{first}, {last}) of a sequence of {end}")
        at = np.arange(first, last, dtype=np.int64)
        pages = np.asarray(self._pages.get(seq, []), np.int64)
        return pages[at // self.cache.page_size] * self.cache.page_size + at % self.cache.page_size

    def drop(self, seq: Hashable) -> None:
        """Gives a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(seq, [])))
        self._length.pop(seq, None)

    def extend(self, new_tokens: Dict[Hashable, int]) -> PagedBatch:
        """Room for ``new_tokens[seq]`` more tokens of each sequence (new ones start empty), and the batch's arrays.
        ``MemoryError`` where the cache has too few free pages; nothing is taken then, nor where the arrays cannot be made."""
        size = self.cache.page_size
        if any(n < 0 for n in new_tokens.values()):
            raise ValueError("a sequence cannot lose tokens")
        want = {s: -(-(self.length(s) + n) // size) - len(self._pages.get(s, [])) for s, n in new_tokens.items()}
        if sum(want.values()) > len(self._free):
            raise MemoryError(f"{sum(want.values())} pages wanted, {len(self._free)} free")
        before = {s: self.length(s) for s in new_tokens}
        known = {s for s in new_tokens if s in self._pages}
        for s, n in new_tokens.items():
            self._pages.setdefault(s, []).extend(self._free.pop() for _ in range(want[s]))
            self._length[s] = before[s] + n
        try:
            return self._batch(new_tokens, before)
        except BaseException:                                  # (no arrays, no step: the pages go back in the order they came)
            for s in reversed(list(new_tokens)):
                for _ in range(want[s]):
                    self._free.append(self._pages[s].pop())
                self._length[s] = before[s]
                if s not in known:
                    del self._pages[s], self._length[s]
            raise

    def _batch(self, new_tokens: Dict[Hashable, int], before: Dict[Hashable, int]) -> PagedBatch:
        seqs = list(new_tokens)
        width = max([len(self._pages[s]) for s in seqs] + [1])
        table = np.zeros((len(seqs), width), np.int32)
        for b, s in enumerate(seqs):
            table[b, : len(self._pages[s])] = self._pages[s]
        lens = np.asarray([self._length[s] for s in seqs], np.int32)
        offsets = np.concatenate([[0], np.cumsum([new_tokens[s] for s in seqs])]).astype(np.int32)
        slots = np.concatenate([self.slots(s, before[s]) for s in seqs] + [np.zeros(0, np.int64)])
        put = DeviceArray.from_host
        return PagedBatch(put(slots), put(table), put(offsets), put(lens), max(new_tokens.values(), default=0),
                          int(lens.max(initial=0)))


def _attend(q_ptr: int, q_token: int, T: int, Hq: int, cache: PagedKVCache, batch: PagedBatch, scale, causal, window, softcap,
            return_lse, out):
    if out not in ("storage", "f32"):
        raise ValueError("out must be 'storage' or 'f32'")
    table, offsets, lens = batch.page_table, batch.q_offsets, batch.kv_lens
    if any(a.dtype != "i32" for a in (table, offsets, lens)) or table.ndim != 2:
        raise ValueError("page_table, q_offsets and kv_lens must be i32, page_table (B, pages)")
    B, D = table.shape[0], cache.head_dim
    if batch.slots is not None and batch.slots.shape != (T,):
        raise ValueError(f"queries of {T} tokens for a batch of {batch.slots.shape[0]}")
    if offsets.shape != (B + 1,) or lens.shape != (B,):
        raise ValueError(f"q_offsets {offsets.shape} and kv_lens {lens.shape} for {B} sequences")
    O = _result((T, Hq, D), "f32" if out == "f32" else cache.dtype)
    L = _result((T, Hq), "f32") if return_lse else None
    strides = (ctypes.c_int64 * 4)(q_token, D, Hq * D, D)
    fn = getattr(_lane.load(), f"tessera_gfx950_paged_attention_{cache.dtype}_dev")
    _lane.check(fn(ctypes.byref(cache.handle), q_ptr, O.address, L.address if L else None, strides, table.address,
                   table.shape[1], offsets.address, lens.address, B, Hq, T, batch.max_q, batch.max_kv,
                   ctypes.c_float(float(scale) if scale is not None else 1.0 / math.sqrt(D)), 1 if causal else 0, int(window),
                   ctypes.c_float(softcap), 0 if out == "f32" else 1, None), "paged_attention")
    return (O, L) if return_lse else O


def paged_attention(Q: DeviceArray, cache: PagedKVCache, batch: PagedBatch, *, scale: Optional[float] = None,
                    causal: bool = True, window: int = 0, logit_softcap: float = 0.0, return_lse: bool = False,
                    out: str = "storage"):
    """Attention of the batch's new tokens ``Q [T, Hq, D]`` over their sequences' keys; returns ``O [T, Hq, D]``
    (``out``: ``"storage"`` or ``"f32"``) and, on request, the log-sum-exp f32 ``[T, Hq]``.  ``causal``, ``window`` and
    ``logit_softcap`` as in :func:`tessera_amd.ops.flash_attn`; a token that sees no key gives 0 and -inf."""
    if Q.dtype != cache.dtype or Q.ndim != 3 or Q.shape[2] != cache.head_dim or Q.shape[1] % cache.num_kv_heads:
        raise ValueError(f"Q must be {cache.dtype} (T, a multiple of {cache.num_kv_heads}, {cache.head_dim}); got {Q.dtype} {Q.shape}")
    T, Hq, D = Q.shape
    return _attend(Q.address, Hq * D, T, Hq, cache, batch, scale, causal, window, logit_softcap, return_lse, out)


def paged_attention_fused_qkv(QKV: DeviceArray, num_q_heads: int, cache: PagedKVCache, batch: PagedBatch, *,
                              scale: Optional[float] = None, causal: bool = True, window: int = 0, logit_softcap: float = 0.0,
                              return_lse: bool = False, out: str = "storage"):
    """The same from the output of one fused projection, ``QKV [T, (Hq + 2 Hkv) * D]``, whose K and V columns
    :meth:`PagedKVCache.write_fused_qkv` has put into the cache: the query columns are read where they lie."""
    width = (num_q_heads + 2 * cache.num_kv_heads) * cache.head_dim
    if QKV.dtype != cache.dtype or QKV.ndim != 2 or QKV.shape[1] != width or num_q_heads % cache.num_kv_heads:
        raise ValueError(f"QKV must be {cache.dtype} (T, {width}), the query heads a multiple of {cache.num_kv_heads}; got "
                         f"{QKV.dtype} {QKV.shape}")
    return _attend(QKV.address, width, QKV.shape[0], num_q_heads, cache, batch, scale, causal, window, logit_softcap, return_lse, out)
