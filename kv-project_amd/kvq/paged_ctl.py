"""The attention router's controller over a ``PagedCache``: prompts and steps of a batch of sequences.

``with routed(PagedCtl(cache, slots)) as ctl: ctl.begin(counts); model(...)`` runs a model whose attention is
registered under ``kvq.register()`` (STRATA_KV.py:495-523) on the slots of the cache: each layer's new keys
and values are appended to its pages, and its queries attend

* over the prompt itself (prompt_attention, exact keys and values) where a sequence begins, whoever else is in the batch,
* over the cache by ``paged_decode`` in steps of a few tokens,
* over the cache's rows by ``rows`` and prompt_attention in steps of many tokens (a further question, a chunk of
  a prompt): the same attention as paged_decode's, with the codes read once rather than once per 16 query rows; or, with
  ``over_pages``, straight over the pages by ``paged_attention``: without the rows' rounding and their memory, and a text that
  neighbouring slots share (forks side by side) once for all of them.

Layer ``module.layer_idx`` of the model is layer ``layer_idx`` of the cache.
"""
from __future__ import annotations

import itertools
from typing import Sequence, Union

import torch

from . import paged
from .paged import PagedPlan, paged_attention
from .pages import PagedCache, paged_decode
from .prompt import PromptPlan, prompt_attention

# Query rows per KV head of a sequence (query heads times new tokens) from which on the rows are read back.  Both ways,
# decode / read back, on an MI355X with 8 KV heads of 128, at 128 and at 256 rows: 16 sequences of 16384 tokens 422 / 525
# and 781 / 587 us, 8 of 2048 49 / 48 and 80 / 57, one of 8192 33 / 38 and 49 / 41 (head_dim 64: 230 / 281 and 444 / 322,
# 27 / 32 and 46 / 37, 20 / 30 and 30 / 32).
MANY_ROWS = 192


class PagedCtl:
    """Sequences in ``slots`` of ``cache``, the rows of the model's batch in that order.  ``over_pages``: steps of many tokens
    attend straight over the pages (the codes as they are, where reading back rounds them to the model's type).  They are many from 33 rows a
    KV head on, where reading back is from 192 on: steps between these leave paged_decode, whose weights have 17 bits, for
    paged_attention's, one number of the model's type as in prompt_attention."""

    def __init__(self, cache: PagedCache, slots: Sequence[int], *, over_pages: bool = False):
        self.cache, self.slots, self.over_pages = cache, [int(s) for s in slots], bool(over_pages)
        self.step = None

    def begin(self, counts: Union[int, Sequence[int]]) -> None:
        """Claim the next step: ``counts`` new tokens of every sequence, or of each one (in a batch padded on the left:
        the last counts[b] tokens of row b are its own).  Once per forward pass, before it: a layer that comes a second time
        in a step is refused, its tokens would take the places of the first ones.  To run a step again on purpose (a pass that
        failed, one in front of a capture) clear ``seen``."""
        n = [int(counts)] * len(self.slots) if isinstance(counts, int) else [int(c) for c in counts]
        if len(n) != len(self.slots):
            raise ValueError("counts must be one number or one per sequence")
        before = [self.cache.length(s) for s in self.slots]
        self.step = None                       # none is left if this one does not fit
        self.step = self.cache.extend(self.slots, n)
        self.counts, self.lens = n, [a + b for a, b in zip(before, n)]
        self.begins, self.runs = ([b for b, c in enumerate(n) if c and bool(before[b]) == held] for held in (False, True))
        self.plans, self.index, self.own = {}, None, None
        self.seen = set()                      # layers that have appended the step

    def _plan(self, Hq: int, which, lens_k) -> PromptPlan:
        key = (Hq, lens_k is None)                            # one for all layers of the step
        if key not in self.plans:
            self.plans[key] = PromptPlan([self.counts[b] for b in which], Hq, self.cache.Hkv, device=self.cache.device,
                                         lens_k=None if lens_k is None else [lens_k[b] for b in which])
        return self.plans[key]

    def _rows_of(self, which, device):
        """The packed rows of some of the sequences: a slice where they lie behind one another."""
        first = [0, *itertools.accumulate(self.counts)]
        parts = [(first[b], first[b + 1]) for b in which]
        if all(x[1] == y[0] for x, y in zip(parts, parts[1:])):
            return slice(parts[0][0], parts[-1][1])
        return torch.cat([torch.arange(*x) for x in parts]).to(device)

    def _packed(self, x: torch.Tensor, T: int) -> torch.Tensor:
        """(B, H, T, d) -> the sequences' own rows (rows, H, d)."""
        x = x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])
        return x if self.index is None else x.index_select(0, self.index)

    def attend(self, module, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask, kwargs):
        """One layer of the step (the controller's part of router_attention): q (B, Hq, T, d), k, v (B, Hkv, T, d) ->
        ((B, T, Hq, d), None).  Rows of padding come out as zeros."""
        if self.step is None:
            raise RuntimeError("PagedCtl: begin() claims the step before the forward pass")
        B, Hq, T, d = q.shape
        if B != len(self.slots) or k.shape[2] != T or T < max(self.counts):
            raise ValueError(f"PagedCtl: a batch of {B} rows of {T} tokens for {len(self.slots)} sequences of up to "
                             f"{max(self.counts)} new tokens")
        if self.index is None and min(self.counts) < T:
            own = torch.arange(T)[None] >= T - torch.tensor(self.counts)[:, None]
            self.index = own.reshape(-1).nonzero()[:, 0].to(q.device)
        scaling = kwargs.get("scaling")
        scaling = module.scaling if scaling is None else scaling
        layer, cache = module.layer_idx, self.cache
        if layer in self.seen:
            raise RuntimeError(f"PagedCtl: layer {layer} has had this step; begin() claims one for each forward pass")
        qp, kp, vp = (self._packed(x, T) for x in (q, k, v))
        cache.append(layer, kp, vp, self.step)
        self.seen.add(layer)
        few = Hq // cache.Hkv * max(self.counts) < (paged.FEW_ROWS + 1 if self.over_pages else MANY_ROWS)
        if not self.runs:
            out = prompt_attention(qp, kp, vp, scaling, self._plan(Hq, self.begins, None))
        elif not self.begins:
            out = paged_decode(qp, scaling, cache, layer, self.step) if few else self._over_rows(qp, scaling, layer)
        else:                                  # each kind of sequence its own way
            if self.own is None:
                self.own = [self._rows_of(which, q.device) for which in (self.begins, self.runs)]
            begins, runs = self.own
            if few:
                out = paged_decode(qp, scaling, cache, layer, self.step)
            else:
                out = torch.empty_like(qp)
                out[runs] = self._over_rows(qp[runs], scaling, layer)
            out[begins] = prompt_attention(qp[begins], kp[begins], vp[begins], scaling, self._plan(Hq, self.begins, None))
        if self.index is None:
            return out.view(B, T, Hq, d), None
        whole = torch.zeros((B * T, Hq, d), dtype=out.dtype, device=out.device)
        whole.index_copy_(0, self.index, out)
        return whole.view(B, T, Hq, d), None

    def _over_rows(self, q: torch.Tensor, scaling: float, layer: int) -> torch.Tensor:
        """The running sequences' rows q over the cache: straight over its pages, or its rows, read back."""
        slots = [self.slots[b] for b in self.runs]
        if self.over_pages:
            key = (q.shape[1], "pages")
            if key not in self.plans:
                self.plans[key] = PagedPlan(self.cache, slots, [self.counts[b] for b in self.runs], q.shape[1])
            return paged_attention(q, scaling, self.cache, layer, self.plans[key])
        k, v = self.cache.rows(layer, slots)
        return prompt_attention(q, k, v, scaling, self._plan(q.shape[1], self.runs, self.lens))
