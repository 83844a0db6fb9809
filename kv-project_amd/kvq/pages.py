"""A KV cache in pages of 8-bit codes, shared by sequences of any lengths, for all layers of a model.

``PagedCache`` holds, per layer, a pool of pages: ``page`` tokens of every KV head as int8 or e4m3 codes with
one float32 scale for the keys and one for the values of each head.  A sequence is a slot: a row of the
page table and the block that is still open, in the model's type.  A block is coded when its last token
comes, so what the cache holds does not depend on how the tokens arrived.  Full pages are never written
again; forked sequences share them by count.

A step: ``step = cache.extend(slots, counts)`` claims room for new tokens of some sequences, once for all
layers; ``cache.append(layer, k, v, step)`` and ``paged_decode(q, scaling, cache, layer, step)`` run per layer.
The page accounts live in host memory (libkvq's kvq_pages_* calls); the kernels read the table and the
step's description on the device.  The reference's caches are dense in the batch (STRATA_KV.py:682-719):
this one has no counterpart there.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .prompt import device_of, rows16

CODES = {"int8": 0, "e4m3": 1}
PAGES = (32, 64, 128)
# Workgroups a decode is split into at most, by head_dim: two and three on each of 256 CUs.  16 sequences at 32k,
# head_dim 128: 197 us with 512, 202 with 768; 48 ragged ones, head_dim 64: 40 with 512, 33 with 768, 34 with 1024.
SPLIT_BLOCKS = {128: 512, 64: 768}
# One on each CU where there are few units of 64 tokens (times KV heads), joined in the same launch: with 256 and with
# 512, at head_dim 128, 2048 of them 13.5 and 18.4 us, 8192 29.4 and 34.8, 16384 55.9 and 55.8.
FEW_BLOCKS, FEW_UNITS = 256, 16384



def _ints(x, what: str) -> np.ndarray:
    a = np.array(x, dtype=np.int64).reshape(-1)
    if a.size == 0:
        raise ValueError(f"{what} must not be empty")
    return a


_Start = C.c_char * 0


def _address(a: np.ndarray) -> int:
    """The address of an array that may be written (a third of the time that ``a.ctypes.data`` takes)."""
    return C.addressof(_Start.from_buffer(a))


class Step:
    """New tokens of some slots: ``rows`` packed rows, slot by slot.  Made by ``PagedCache.extend``."""

    __slots__ = ("cache", "slots", "counts", "made", "rows", "items", "splits", "run_tokens", "split_tokens", "joins", "fronts", "shares",
                 "desc", "ptr", "host", "generation", "pools", "stamp", "streams")


class PagedCache:
    """``layers`` layers of ``pages`` pages for ``slots`` sequences of at most ``max_tokens`` tokens: ``Hkv`` KV heads of
    head_dim ``d`` (64 or 128), blocks of ``page`` tokens (32, 64 or 128) held as ``code`` ("int8" or "e4m3"), rows of
    ``dtype`` (bf16 or fp16).

    Calls on one cache run in the order in which they are made: on one stream, or on streams that wait for each other
    (the accounts of slots and pages are on the host and change at once; not thread-safe).  append and paged_decode may be
    captured in a graph, for steps that ``extend(..., into=step)`` writes in front of each replay; the calls that change
    slots or pages may not.  Memory that is dropped (a step's, the pools' by resize(), the cache's) is kept until the
    streams that the calls were made on are done with it.  A captured graph reads and writes the cache's memory and its
    step's: both have to live as long as it is replayed, and resize() ends its use."""

    def __init__(self, layers: int, slots: int, pages: int, max_tokens: int, Hkv: int, d: int, *, page: int = 64,
                 code: str = "int8", dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(layers, slots, pages, max_tokens, Hkv) < 1:
            raise ValueError("a cache needs at least one layer, slot, page, token and KV head")
        if d not in (64, 128):
            raise _lib.KVQError(f"PagedCache: head_dim must be 64 or 128 (got {d})")
        if page not in PAGES:
            raise ValueError(f"page must be one of {PAGES}")
        if code not in CODES:
            raise ValueError(f"code must be one of {tuple(CODES)}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("PagedCache holds bf16 or fp16 rows")
        if max(pages, max_tokens, slots) >= 1 << 31 or layers * Hkv >= 65536:
            raise ValueError("too many pages, tokens, slots or heads")
        self.device = device_of(device)
        self.layers, self.slots, self.pages, self.max_tokens = int(layers), int(slots), int(pages), int(max_tokens)
        self.Hkv, self.d, self.page, self.code, self.dtype = int(Hkv), int(d), int(page), code, dtype
        self.max_blocks = -(-self.max_tokens // self.page)
        self._lens = np.zeros(self.slots, dtype=np.int64)
        self._table = np.zeros((self.slots, self.max_blocks), dtype=np.int32)
        self._open = np.zeros(self.slots, dtype=np.uint8)
        self._refs = np.zeros(self.pages, dtype=np.int32)
        self._account = np.array([self.pages, 0], dtype=np.int64)   # free pages, none of them below
        self._generation = 0                   # of the pages' places
        self._pools = 0                        # of the pools
        self._stamp = 0                        # of the slots' lengths
        self._touched = np.zeros(self.slots, dtype=np.int64)        # the stamp when a slot took tokens or was emptied
        self._away = None                      # the DeviceAccounts that have the accounts meanwhile
        self.table = torch.zeros((self.slots, self.max_blocks), dtype=torch.int32, device=self.device)
        self.kc, self.vc, self.sc = self._pool(self.pages)
        rows = (self.layers, self.slots, 2, self.Hkv, self.page * self.d)
        self.k_open = torch.zeros(rows, dtype=dtype, device=self.device)     # token major, as a page's keys
        self.v_open = torch.zeros(rows, dtype=dtype, device=self.device)     # channel major, as a page's values
        # counters of the decodes that join their parts in one launch: zeros between calls
        self._counters = torch.zeros((self.layers, self.slots, self.Hkv, 32), dtype=torch.int32, device=self.device)
        self._tickets = [self._counters[l].data_ptr() for l in range(self.layers)]
        self._set_addresses()

    def _pool(self, pages: int):
        new = lambda *s, dt=torch.int8: torch.empty((self.layers, pages, self.Hkv, *s), dtype=dt, device=self.device)
        return new(self.page, self.d), new(self.d, self.page), new(2, dt=torch.float32)

    def _set_addresses(self) -> None:
        """Of each layer's codes, scales and open blocks; what every call passes.  Called where the pools are allocated."""
        self._streams = {_lib.stream_of(self.table)}     # that the pools and the other memory belong to, or are recorded for
        self._host = tuple(x.ctypes.data for x in (self._lens, self._table, self._refs, self._open, self._account))
        self._index, self._type = self.device.index, _lib.DTYPE_CODE[self.dtype]
        self._fixed = (self.table.data_ptr(), self.max_blocks, self.Hkv, self.d, self.page, CODES[self.code])
        parts = [(x.data_ptr(), x.stride(0) * x.element_size()) for x in (self.kc, self.vc, self.sc, self.k_open, self.v_open)]
        self._at = [tuple(p + l * step for p, step in parts) for l in range(self.layers)]

    def _use(self, stream: int, step: Optional[Step] = None) -> None:
        """The current stream, ``stream``, reads and writes the memory of the cache and of ``step``: what is dropped before it is
        done is not given out again until then.  (What a graph is captured with has to outlive it in any case.)"""
        if torch.cuda.is_current_stream_capturing():
            return
        current = torch.cuda.current_stream(self.device)
        if stream not in self._streams:
            for x in (self.table, self.kc, self.vc, self.sc, self.k_open, self.v_open, self._counters):
                x.record_stream(current)
            self._streams.add(stream)
        if step is not None and stream not in step.streams:
            step.desc.record_stream(current)
            step.streams.add(stream)

    # ---- what is held ------------------------------------------------------------------------

    def at_home(self) -> None:
        """Refused while the accounts are on the device."""
        if self._away is not None:
            raise _lib.KVQError("the cache's accounts are on the device: DeviceAccounts.close() hands them back")

    @property
    def lengths(self) -> List[int]:
        """Tokens of each slot."""
        self.at_home()
        return self._lens.tolist()

    def length(self, slot: int) -> int:
        """Tokens of one slot."""
        self.at_home()
        if not 0 <= slot < self.slots:
            raise IndexError(f"no slot {slot} (of {self.slots})")
        return int(self._lens[slot])

    @property
    def free_pages(self) -> int:
        self.at_home()
        return int(self._account[0])

    def codes(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The pools' key and value codes, (layers, pages, Hkv, page, d) views (the values' tokens vary fastest)."""
        dt = torch.int8 if self.code == "int8" else torch.float8_e4m3fn
        return self.kc.view(dt), self.vc.view(dt).transpose(-1, -2)

    def scales(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The pools' key and value scales, (layers, pages, Hkv) float32 views."""
        return self.sc[..., 0], self.sc[..., 1]

    def bytes_per_token(self) -> float:
        """Bytes a full block holds per token, all layers."""
        return self.layers * self.Hkv * (2.0 * self.d + 8.0 / self.page)

    # ---- steps -------------------------------------------------------------------------------

    def extend(self, slots: Sequence[int], counts: Sequence[int], *, into: Optional[Step] = None) -> Step:
        """Claim room for counts[i] more tokens (or none) of slots[i] (each slot once): the lowest free page for each
        block that gets full.  Raises KVQError ("decode buffer exhausted") and changes nothing when a slot or the pool is
        full.  ``into``: a step of the same counts whose description is rewritten in place, so that a
        captured graph of its append and decode runs the new step when it is replayed; refused for a step from before a
        resize(), whose graphs hold pools that are gone."""
        if self._away is not None:
            self.at_home()
        s, c = _ints(slots, "slots"), _ints(counts, "counts")
        if s.shape != c.shape:
            raise ValueError("slots and counts must have the same length")
        n, pc = s.size, _address(c)
        lib, stream = _lib.load(), _lib.stream_of(self.table)
        if into is None:
            words = lib.kvq_pages_step_words(self.page, pc, n)
            if words < 0:
                raise ValueError("counts must not be negative, and below 2^31")
            if words > 32 * n + 32 + n * (self.max_blocks + 1):         # before memory is taken for its description
                raise _lib.KVQError(f"decode buffer exhausted: a slot holds {self.max_tokens} tokens, {int(c.max())} more asked for")
            st = Step()
            st.cache, st.pools = self, self._pools
            st.host = np.empty(words, dtype=np.int32)
            st.desc = self.table.new_empty(words)
            st.ptr, st.streams = st.desc.data_ptr(), {stream}
            st.splits = max(n, -(-SPLIT_BLOCKS[self.d] // self.Hkv))
            st.run_tokens = st.split_tokens = 1 << 31
            few = (-(-FEW_BLOCKS // self.Hkv), FEW_UNITS // self.Hkv)
        else:
            st = into
            if st.cache is not self:
                raise ValueError("a step is rewritten by its own cache only")
            if st.host is None or not np.array_equal(st.counts, c):
                raise ValueError("a step is rewritten for the same counts only")
            if st.pools != self._pools:
                raise ValueError("a step from before resize() is not rewritten: graphs captured with it hold the old pools")
            few = (0, 0)
            if stream not in st.streams:
                self._use(stream, st)
        # a captured decode joins shared fronts only if it was captured with some
        run_tokens = st.run_tokens if into is None or st.shares else 0
        _lib.call_on(self.device, "kvq_pages_extend", *self._host, self.slots, self.pages, self.max_blocks, self.page,
                     self.max_tokens, _address(s), pc, n, st.splits, *few, run_tokens, st.split_tokens,
                     _address(st.host), st.host.size, st.ptr, stream)
        head = st.host[:11].tolist()
        if into is None:
            # what later steps written into this one keep to: without shared fronts any of them does
            st.splits, st.run_tokens, st.joins = max(1, head[2]), head[6], head[10]
            st.split_tokens = max(head[7], st.splits * head[5])
            st.items, st.rows = st.host.size - 32 * n - 32, int(st.host[8 * n + 15])
        st.fronts = head[8] > n
        if into is None:
            st.shares = st.fronts
        self._stamp += 1
        self._touched[s[c > 0] if 0 in counts else s] = self._stamp
        st.slots, st.counts, st.generation, st.made, st.stamp = s, c, self._generation, self._stamp, self._stamp
        return st

    def check_step(self, step: Step, what: str) -> None:
        """A step describes its slots only until they take more tokens or are freed."""
        if step.cache is not self:
            raise ValueError(f"{what}: the step is of another cache")
        if step.stamp != self._stamp:
            if (self._touched[step.slots] > step.made).any():
                raise ValueError(f"{what}: the step's slots have changed since it was made")
            step.stamp = self._stamp           # what changed were other slots

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, step: Step) -> None:
        """The step's new rows k, v (rows, Hkv, d) of one layer, slot by slot: full blocks to codes, the rest to the open
        blocks.  Every layer appends every step, before the slots take the next one.  Running it again writes the same."""
        if not 0 <= layer < self.layers:
            raise IndexError(f"no layer {layer} (of {self.layers})")
        shape = (step.rows, self.Hkv, self.d)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"append: k {tuple(k.shape)} and v {tuple(v.shape)} must be {shape}")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise TypeError("appended rows must have the cache's dtype")
        if k.get_device() != self._index or v.get_device() != self._index:
            _lib.require_gpu(k, v)
            raise ValueError(f"append: the cache is on {self.device}")
        if step.cache is not self or step.stamp != self._stamp:
            self.check_step(step, "append")
        if step.generation != self._generation:
            raise ValueError("append: the pages have moved since the step was made")
        if step.rows == 0:
            return
        (k, kp, kt, kh), (v, vp, vt, vh) = rows16(k), rows16(v)
        stream = _lib.stream_of(k)
        if stream not in step.streams or stream not in self._streams:
            self._use(stream, step)
        _lib.call_on(self.device, "kvq_pages_append", kp, kt, kh, vp, vt, vh, self._type, step.ptr, step.items,
                     *self._fixed, *self._at[layer], stream)

    def rows(self, layer: int, slots: Sequence[int]) -> Tuple[torch.Tensor, torch.Tensor]:
        """All tokens of the slots, one behind the other, as dense rows k, v (tokens, Hkv, d): code times scale, rounded
        once, and the open blocks as they are.  With prompt_attention this is the attention of many new tokens."""
        if not 0 <= layer < self.layers:
            raise IndexError(f"no layer {layer} (of {self.layers})")
        self.at_home()
        s = _ints(slots, "slots")
        total = sum(self._lens.take(s, mode="clip").tolist())
        out = self.k_open.new_empty((2, total, self.Hkv, self.d))
        k, v = out.unbind(0)
        stream = _lib.stream_of(out)
        if stream not in self._streams:
            self._use(stream)
        _lib.call_on(self.device, "kvq_pages_rows", self._host[0], self._host[3], self.slots, _address(s), s.size,
                     *self._fixed, self._type, *self._at[layer], k.data_ptr(), v.data_ptr(), k.numel(), stream)
        return k, v

    # ---- sequences and pages -----------------------------------------------------------------

    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Empty slots dst[i] become continuations of src[i]: they share its pages and get copies of its open block, in all
        layers.  Call it when every layer has appended its steps."""
        self.at_home()
        s, t = _ints(src, "src"), _ints(dst, "dst")
        if s.shape != t.shape:
            raise ValueError("src and dst must have the same length")
        stream = _lib.stream_of(self.table)
        if stream not in self._streams:
            self._use(stream)
        _lib.call_on(self.device, "kvq_pages_fork", *self._host[:4], self.slots, self.max_blocks, self.page, _address(s),
                     _address(t), s.size, self.layers, self.Hkv, self.d, self.table.data_ptr(), self.k_open.data_ptr(), self.v_open.data_ptr(),
                     stream)
        self._stamp += 1
        self._touched[t] = self._stamp

    def free(self, slots: Sequence[int]) -> None:
        """Empty the slots; pages that no other sequence shares become free."""
        self.at_home()
        s = _ints(slots, "slots")
        _lib.call("kvq_pages_free", *self._host, self.slots, self.max_blocks, self.page, _address(s), s.size)
        self._stamp += 1
        self._touched[s] = self._stamp

    def compact(self) -> int:
        """Move the pages at the end of the pool to the free places below, in order, so that the pages in use are the
        first ones; returns their number.  In place: only the moved pages are read and written."""
        used = self.pages - self.free_pages
        self._move(used, None)
        return used

    def resize(self, pages: int) -> None:
        """Give the pool ``pages`` pages: those beyond the new end move to the lowest free places, in order, the others
        keep theirs.  New pools are allocated beside the old ones, whose memory is then given back: graphs captured before may
        not be replayed any more, and their steps not be rewritten."""
        pages = int(pages)
        if pages < max(1, self.pages - self.free_pages):
            raise ValueError(f"{self.pages - self.free_pages} pages are in use")
        if pages >= 1 << 31:
            raise ValueError("too many pages")
        self._move(pages, self._pool(pages))

    def _move(self, end: int, pool) -> None:
        """Pages from ``end`` on to the lowest free places; with ``pool``, every page in use into that one of ``end`` pages."""
        pages = self.pages if pool is None else end
        refs = self._refs if pool is None else np.empty(pages, dtype=np.int32)
        place = np.empty(self.pages, dtype=np.int32)
        src, stream = (self.kc, self.vc, self.sc), _lib.stream_of(self.table)
        if stream not in self._streams:
            self._use(stream)
        _lib.call_on(self.device, "kvq_pages_move", *self._host[:3], _address(refs), self._host[4], self.slots, self.pages,
                     pages, end, self.max_blocks, self.page, _address(place), self.layers, self.Hkv, self.d,
                     *[x.data_ptr() for x in src], *[x.data_ptr() for x in (src if pool is None else pool)], self._fixed[0], stream)
        if pool is not None:
            (self.kc, self.vc, self.sc), self.pages, self._refs = pool, pages, refs
            self._pools += 1
            self._set_addresses()
        self._generation += 1


def paged_workspace_floats(step: Step, Hq: int, Hkv: int, d: int) -> int:
    """Float32 scratch of a decode of this step, and of those that are written into it: none where every sequence is one
    split item."""
    if not step.joins:
        return 0
    n = _lib.load().kvq_paged_decode_workspace(step.split_tokens, Hkv, Hq // Hkv, d)
    if n < 0:
        raise _lib.KVQError("kvq_paged_decode_workspace rejected the shape")
    return n


def paged_decode(q: torch.Tensor, scaling: float, cache: PagedCache, layer: int, step: Step, *,
                 out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the step's query rows q (rows, Hq, d), slot by slot, over the cache; returns (rows, Hq, d).  Query i of
    a slot's new tokens sees every token up to its own.  Pages that neighbouring slots of the step share (forks of one
    sequence, named side by side) are read once for all of them.  Meant for a few tokens per slot (16 rows = query
    heads of a KV head times tokens go over the keys together); for many, ``cache.rows`` and prompt_attention."""
    if not 0 <= layer < cache.layers:
        raise IndexError(f"no layer {layer} (of {cache.layers})")
    shape, Hkv, d = q.shape, cache.Hkv, cache.d
    if len(shape) != 3 or shape[0] != step.rows or shape[2] != d or shape[1] < 1 or shape[1] % Hkv:
        raise ValueError(f"paged_decode: q {tuple(shape)} does not match the step ({step.rows} rows) and the cache "
                         f"({Hkv} KV heads, head_dim {d})")
    if q.dtype != cache.dtype:
        raise TypeError("q must have the cache's dtype")
    if q.get_device() != cache._index:
        _lib.require_gpu(q)
        raise ValueError(f"paged_decode: the cache is on {cache.device}")
    if step.cache is not cache or step.stamp != cache._stamp:
        cache.check_step(step, "paged_decode")
    q, qp, qt, qh = rows16(q)
    Hq, device, stream = shape[1], cache.device, _lib.stream_of(q)
    if out is None:
        # a step of counts that the host does not know may leave rows out
        new = torch.empty_like if step.host is not None else torch.zeros_like
        out = new(q, memory_format=torch.contiguous_format)
    else:
        _lib.out_or_new(out, shape, cache.dtype, device, "paged_decode")
    if step.rows == 0:
        return out
    if workspace is None:
        workspace = cache.sc.new_empty(paged_workspace_floats(step, Hq, Hkv, d))
    elif workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.device != device:
        raise ValueError("workspace must be contiguous float32 on the cache's device")
    if stream not in step.streams or stream not in cache._streams:
        cache._use(stream, step)
    table, max_blocks, _, _, page, code = cache._fixed
    _lib.call_on(device, "kvq_paged_decode", qp, qt, qh, cache._type, step.rows, Hq, Hkv, d, float(scaling), step.ptr,
                 step.slots.size, step.splits, step.run_tokens, step.split_tokens, step.joins, table, max_blocks, page,
                 code, *cache._at[layer], out.data_ptr(), workspace.data_ptr(), workspace.numel(),
                 None if step.shares else cache._tickets[layer], stream)
    return out
