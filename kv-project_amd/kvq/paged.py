"""Attention of many query rows straight over a ``PagedCache``.

``paged_decode`` is for a step's few new tokens.  Here the rows may be many, and any: the last tokens of slots (a chunk
of a prompt, a question behind a text), whose text may be shared, or, with ``causal=False``, rows of other sequences that see
every token of a slot (cross attention to an encoder's states, held in a cache of their own).  ``PagedPlan`` is built once
from the slots and counts (on the host) and serves every layer of the step.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from .pages import FEW_BLOCKS, FEW_UNITS, SPLIT_BLOCKS, PagedCache, _address
from .prompt import MAX_REP, rows16

# Rows (query heads of a KV head times tokens) of a sequence up to which paged_decode's kernels take them, 16 at a time, and in
# fours of these for neighbours over a shared text.  Theirs / those of tiles of 128 rows, 8 KV heads of 128: 16 sequences of
# 16384 tokens with 32 rows 128 / 153 us, with 48 169 / 154; 64 of 1000 37 / 41 and 48 / 42; 8 behind a text of 8192, 16 rows each 23 / 25,
# 32 each 35 / 28.
FEW_ROWS = 32
# Beside sequences of many rows those of few have launches of their own from this many units (64 tokens of a KV head) on: 10 us of
# the chip's tiles.
FEW_WORK = 2048


class PagedPlan:
    """The work of an attention of packed rows over ``cache``: counts[i] rows (or none) for slots[i], behind one another, ``Hq``
    query heads each.  Causal: the rows are the slot's last tokens, and each sees those up to its own.  Otherwise every row sees
    all tokens of the slot; rows of a slot without tokens get zeros.

    Pages that neighbours share in front (forks of one sequence, named side by side) are read once for all of them where that saves
    work, and a slot named several times in a row without ``causal`` is read once altogether.  A plan describes its slots until they
    take more tokens or are freed; one that is dropped is kept until the streams of its calls are done with it, and it has to
    live as long as a graph captured with it is replayed."""

    def __init__(self, cache: PagedCache, slots: Sequence[int], counts: Sequence[int], Hq: int, *, causal: bool = True):
        cache.at_home()
        s, c = (np.array(x, dtype=np.int64).reshape(-1) for x in (slots, counts))
        if s.size == 0 or s.shape != c.shape:
            raise ValueError("slots and counts must have the same length, one at least")
        if Hq < 1 or Hq % cache.Hkv or Hq // cache.Hkv > MAX_REP:
            raise ValueError(f"{Hq} query heads over {cache.Hkv} KV heads: the quotient must be whole and at most {MAX_REP}")
        self.cache, self.Hq, self.causal = cache, int(Hq), bool(causal)
        self.slots, self.counts = s, c
        lens, table, _, open_, _ = cache._host
        info = np.zeros(12, dtype=np.int64)
        args = (lens, table, open_, cache.slots, cache.max_blocks, cache.page, _address(s), _address(c), s.size,
                self.Hq // cache.Hkv, cache.Hkv, cache.d, int(self.causal), FEW_ROWS, FEW_WORK, -(-SPLIT_BLOCKS[cache.d] // cache.Hkv),
                -(-FEW_BLOCKS // cache.Hkv), FEW_UNITS // cache.Hkv)
        words = np.empty(2048, dtype=np.int32)
        _lib.call("kvq_paged_plan", *args, _address(words), words.size, _address(info))
        many = 12 * int(info[0]) + 8 * int(info[1])
        need = many + int(info[4])
        if need > words.size:
            words = np.empty(need, dtype=np.int32)
            _lib.call("kvq_paged_plan", *args, _address(words), words.size, _address(info))
        self.rows = int(c.sum())
        self.items, self.merges, self.parts, self.waves, _, self.sequences, *self._few, self._joins, fronts, self._most_parts = info.tolist()
        self.words = torch.from_numpy(words[:max(need, 1)]).to(cache.device)
        self._at = (self.words.data_ptr(), self.words.data_ptr() + 4 * many)
        lib = _lib.load()
        self._floats = lib.kvq_paged_attention_workspace(self.parts, self.waves, cache.Hkv, cache.d) if self.parts else 0
        self._few_floats = 0
        if self._joins:
            self._few_floats = lib.kvq_paged_decode_workspace(self._few[2], cache.Hkv, self.Hq // cache.Hkv, cache.d)
        # a slot's tickets are one run's
        named = s[c > 0]
        if not causal:
            named = named[np.append(True, named[1:] != named[:-1])] if named.size else named
        self._tickets = not fronts and np.unique(named).size == named.size
        self._stamp = cache._stamp
        self._streams = {_lib.stream_of(self.words)}     # that the words belong to, or are recorded for

    def check(self) -> None:
        """Refused once a slot has taken tokens or was emptied."""
        cache = self.cache
        if self._stamp != cache._stamp:
            if (cache._touched[self.slots] > self._stamp).any():
                raise ValueError("paged_attention: the plan's slots have changed since it was made")

    def workspace_floats(self) -> int:
        """Float32 scratch of a call: none where nothing is cut along the tokens."""
        return self._floats + self._few_floats


def paged_attention(q: torch.Tensor, scaling: float, cache: PagedCache, layer: int, plan: PagedPlan, *,
                    out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the plan's packed rows q (rows, Hq, d) over one layer of the cache; returns (rows, Hq, d).  The codes go into
    the products as they are and their scales in float32; what a row does not see changes nothing, whatever it holds.  Rows beyond a few
    (FEW_ROWS of a sequence) weigh with one number of the model's type, rounded once (half a step: bf16 2^-8, fp16 2^-11 of a weight, which is
    summed as it was rounded), where paged_decode's few rows have two of them (2^-17): the same row differs by that between a call of
    32 rows a KV head and one of 33.  Forward only, as the decodes: no gradient is recorded.

    Value blocks of one sequence may lie far apart in size.  Of two pages of 32 tokens side by side (blocks 2 i and 2 i + 1) a token of the
    smaller one's is off by up to 2^-28 of the larger one's largest value in fp16, and by 2^-100 of the largest that the row sees in bf16."""
    if not 0 <= layer < cache.layers:
        raise IndexError(f"no layer {layer} (of {cache.layers})")
    if plan.cache is not cache:
        raise ValueError("paged_attention: the plan is of another cache")
    shape = q.shape
    if shape != (plan.rows, plan.Hq, cache.d):
        raise ValueError(f"paged_attention: q {tuple(shape)} does not match the plan ({plan.rows} rows of {plan.Hq} heads) and the "
                         f"cache (head_dim {cache.d})")
    if q.dtype != cache.dtype:
        raise TypeError("q must have the cache's dtype")
    if q.get_device() != cache._index:
        _lib.require_gpu(q)
        raise ValueError(f"paged_attention: the cache is on {cache.device}")
    if plan._stamp != cache._stamp:
        plan.check()
    device = cache.device
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _lib.out_or_new(out, shape, cache.dtype, device, "paged_attention")
    if plan.rows == 0:
        return out
    q, qp, qt, qh = rows16(q)
    stream, floats = _lib.stream_of(q), plan._floats + plan._few_floats
    ws = None
    if workspace is None:
        if floats:
            workspace = cache.sc.new_empty(floats)
    elif workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.device != device:
        raise ValueError("workspace must be contiguous float32 on the cache's device")
    elif workspace.numel() < floats:
        raise ValueError(f"a workspace of {workspace.numel()} floats, {floats} needed")
    if (stream not in cache._streams or stream not in plan._streams) and not torch.cuda.is_current_stream_capturing():
        cache._use(stream)
        if stream not in plan._streams:
            plan.words.record_stream(torch.cuda.current_stream(device))
            plan._streams.add(stream)
    table, max_blocks, Hkv, d, page, code = cache._fixed
    at, few = plan._at
    if floats:
        ws = workspace.data_ptr()
    if plan.items:
        _lib.call_on(device, "kvq_paged_attention", qp, qt, qh, cache._type, plan.Hq, Hkv, d, float(scaling), at,
                     plan.items, plan.merges, plan.parts, plan._most_parts, plan.waves, table, max_blocks, page, code, *cache._at[layer], out.data_ptr(),
                     ws, plan._floats, stream)
    if plan.sequences:
        _lib.call_on(device, "kvq_paged_decode_held", qp, qt, qh, cache._type, plan.rows, plan.Hq, Hkv, d, float(scaling), few,
                     plan.sequences, *plan._few, plan._joins, table, max_blocks, page, code, *cache._at[layer], out.data_ptr(),
                     ws + 4 * plan._floats if plan._few_floats else None, plan._few_floats, cache._tickets[layer] if plan._tickets else None, int(not plan.causal), stream)
    return out
