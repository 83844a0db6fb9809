"""A ``PagedCache``'s accounts in device memory: page tables and slot maps from lengths that only the GPU knows.

On the host a step's counts have to be known when ``PagedCache.extend`` is called.  Where they are decided on the GPU (a
sequence that has ended takes nothing, a draft was cut short, the next request's prompt), ``DeviceAccounts`` keeps the
accounts there: ``extend`` and ``free`` are launches that read counts and lengths from device memory, may be captured in a
graph together with ``append`` and ``paged_decode``, and never wait for the host.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .pages import FEW_BLOCKS, FEW_UNITS, SPLIT_BLOCKS, PagedCache, Step, _ints


class DeviceStep(Step):
    """Up to ``most`` new tokens of some slots; made by ``DeviceAccounts.step``.  The rows of the i-th slot are i * most .., the first
    counts[i] of them are its own.  On the device, as of the last ``extend``: ``positions`` (rows,) int32, a row's place in
    its sequence, -1 for a row that is none's; ``places`` (rows,) int64, page * cache.page + offset of a row whose block is full,
    -1 for the others (they lie in the open block)."""

    __slots__ = ("most", "words", "slots_at", "scratch_at", "positions", "places")


class DeviceAccounts:
    """Takes the cache's accounts to the device; until ``close`` hands them back, the cache's own calls that need them (extend, rows,
    fork, free, compact, resize, its lengths, plans) are refused, and so are steps and plans that were made before.  Calls run in the
    order in which they are made, as the cache's do; what a captured graph reads and writes (these accounts, the cache, its steps)
    has to live as long as it is replayed, and graphs of extend and free are not replayed after ``close``.

    ``lengths`` (slots,) int32 is each slot's tokens, ``free_pages`` and ``refused`` () int32 the free pages and the steps that did not
    fit, all on the device."""

    def __init__(self, cache: PagedCache):
        cache.at_home()
        self.cache = cache
        n, p = cache.slots, cache.pages
        state = np.empty(2 * n + p + 4, dtype=np.int32)
        state[:n], state[n:2 * n], state[2 * n:2 * n + p] = cache._lens, cache._open & 1, cache._refs
        state[2 * n + p:] = [*cache._account, 0, 0]
        # entries behind a slot's pages are stale on both sides
        table = np.where(np.arange(cache.max_blocks)[None] < (cache._lens // cache.page)[:, None], cache._table, 0)
        self._state = torch.from_numpy(state).to(cache.device)
        cache.table.copy_(torch.from_numpy(table))
        self.lengths, self._open, self._refs, account = self._state.split([n, n, p, 4])
        self.free_pages, self.refused = account[0], account[2]
        self._at = tuple(x.data_ptr() for x in (self.lengths, self._refs, self._open, account))
        stream = _lib.stream_of(self._state)
        self._streams = {stream}
        cache._use(stream)
        cache._away = self
        self._changed(slice(None))

    def _changed(self, slots, step: Optional[DeviceStep] = None) -> None:
        """Steps and plans over these slots from before are refused."""
        cache = self.cache
        cache._stamp += 1
        cache._touched[slots] = cache._stamp
        if step is not None:
            step.made = step.stamp = cache._stamp

    def _mine(self) -> None:
        if self.cache._away is not self:
            raise _lib.KVQError("these accounts were handed back to the host")

    def _use(self, step: DeviceStep) -> int:
        stream = _lib.stream_of(self._state)
        if (stream not in self._streams or stream not in step.streams) and not torch.cuda.is_current_stream_capturing():
            self.cache._use(stream, step)
            self._state.record_stream(torch.cuda.current_stream(self.cache.device))
            self._streams.add(stream)
        return stream

    def step(self, slots: Sequence[int], most: int) -> DeviceStep:
        """A step of up to ``most`` tokens of each of ``slots`` (each once).  It describes nothing until ``extend``; it may be extended
        any number of times, and several steps of the same slots may take turns."""
        self._mine()
        cache, s, most = self.cache, _ints(slots, "slots"), int(most)
        n = s.size
        if s.min() < 0 or s.max() >= cache.slots:
            raise _lib.KVQError(f"no slot {int(s.min()) if s.min() < 0 else int(s.max())} (of {cache.slots})")
        if np.unique(s).size != n:
            raise _lib.KVQError("a slot is named twice")
        words = _lib.load().kvq_tables_step_words(cache.page, n, most)
        if words < 0:
            raise ValueError("most must be positive, and the step's rows below 2^31")
        if most > cache.max_tokens:
            raise _lib.KVQError(f"a slot holds {cache.max_tokens} tokens, a step of {most} asked for")
        st = DeviceStep()
        st.cache, st.slots, st.counts, st.most, st.words = cache, s, np.full(n, most, dtype=np.int64), most, words
        st.rows = n * most
        st.items = words - 32 * n - 32
        few = n * -(-cache.max_tokens // 64) <= FEW_UNITS // cache.Hkv
        st.splits = max(n, -(-(FEW_BLOCKS if few else SPLIT_BLOCKS[cache.d]) // cache.Hkv))
        st.run_tokens, st.split_tokens, st.joins, st.fronts, st.shares, st.host = most, st.splits * most, 1, False, False, None
        # the description, its new pages, slots, positions and places, in one piece of memory
        scratch = words
        slots_at = scratch + n + st.items
        positions = slots_at + n
        places = positions + st.rows
        places += places % 2
        memory = np.zeros(places + 2 * st.rows, dtype=np.int32)
        memory[slots_at:slots_at + n] = s
        memory[positions:] = -1
        st.desc = torch.from_numpy(memory).to(cache.device)
        st.ptr, st.streams = st.desc.data_ptr(), {_lib.stream_of(st.desc)}
        st.scratch_at, st.slots_at = st.ptr + 4 * scratch, st.ptr + 4 * slots_at
        st.positions, st.places = st.desc[positions:positions + st.rows], st.desc[places:].view(torch.int64)
        st.generation, st.pools = cache._generation, cache._pools
        st.made = st.stamp = cache._stamp
        return st

    def extend(self, step: DeviceStep, counts: torch.Tensor) -> None:
        """Claim counts[i] tokens (int32 on the device, 0 .. step.most) for the step's slots: the lowest free page for each block that
        gets full, in order, as ``PagedCache.extend``.  A step that does not fit (a count out of range, a full slot, too few pages)
        changes no slot, describes no tokens, and adds one to ``refused``, for which ``close`` raises."""
        self._mine()
        cache = self.cache
        if step.cache is not cache or not isinstance(step, DeviceStep) or step.generation != cache._generation:
            raise ValueError("extend: the step is of other accounts")
        if counts.dtype != torch.int32 or counts.shape != step.slots.shape or not counts.is_contiguous():
            raise ValueError(f"counts must be {step.slots.size} contiguous int32")
        if counts.get_device() != cache._index:
            _lib.require_gpu(counts)
            raise ValueError(f"extend: the cache is on {cache.device}")
        stream = self._use(step)
        lens, refs, open_, account = self._at
        _lib.call_on(cache.device, "kvq_tables_extend", step.slots_at, counts.data_ptr(), step.slots.size, step.most, cache.page,
                     cache.max_tokens, cache.pages, cache.max_blocks, step.splits, lens, refs, open_, account, cache._fixed[0], step.ptr,
                     step.words, step.scratch_at, step.slots.size + step.items, step.positions.data_ptr(), step.places.data_ptr(), stream)
        self._changed(step.slots, step)

    def free(self, step: DeviceStep, which: Optional[torch.Tensor] = None) -> None:
        """Empty the step's slots, or those where ``which`` (bool on the device) is true; pages that no other slot shares become free.
        The step then waits for its next ``extend``."""
        self._mine()
        cache = self.cache
        if step.cache is not cache or not isinstance(step, DeviceStep) or step.generation != cache._generation:
            raise ValueError("free: the step is of other accounts")
        at = None
        if which is not None:
            if which.dtype != torch.bool or which.shape != step.slots.shape or not which.is_contiguous():
                raise ValueError(f"which must be {step.slots.size} contiguous bool")
            if which.get_device() != cache._index:
                _lib.require_gpu(which)
                raise ValueError(f"free: the cache is on {cache.device}")
            at = which.data_ptr()
        stream = self._use(step)
        lens, refs, open_, account = self._at
        _lib.call_on(cache.device, "kvq_tables_free", step.slots_at, at, step.slots.size, cache.page, cache.max_blocks, lens, refs, open_,
                     account, cache._fixed[0], stream)
        self._changed(step.slots)

    def close(self) -> None:
        """Hand the accounts back to the host (waits for the GPU).  Raises KVQError, with the accounts handed back, where steps had been
        refused."""
        self._mine()
        cache = self.cache
        n, p = cache.slots, cache.pages
        stream = _lib.stream_of(self._state)
        if stream not in self._streams:
            cache._use(stream)
            self._state.record_stream(torch.cuda.current_stream(cache.device))
        state, table = self._state.cpu().numpy(), cache.table.cpu().numpy()
        cache._lens[:], cache._open[:], cache._refs[:] = state[:n], state[n:2 * n], state[2 * n:2 * n + p]
        cache._table[:] = table
        cache._account[:] = state[2 * n + p:2 * n + p + 2]
        cache._away = None
        self._changed(slice(None))
        refused = int(state[2 * n + p + 2])
        if refused:
            raise _lib.KVQError(f"decode buffer exhausted: {refused} steps did not fit and were left out")

    def __enter__(self) -> "DeviceAccounts":
        return self

    def __exit__(self, kind, *_) -> None:
        if self.cache._away is self:
            try:
                self.close()
            except _lib.KVQError:
                if kind is None:               # not over the error that ended the block
                    raise
