"""Attention over whole prompts: packed sequences of any lengths, grouped heads.

The reference leaves a prompt's attention to SDPA over a dense batch (STRATA_KV.py:499-504); here the
sequences of a batch lie behind one another, (rows, heads, head_dim), with no padding, and a chunk of a
prompt may attend over what is there of it already.  ``PromptPlan`` is built once from the lengths (on the
host) and serves every layer of the step.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib

MAX_REP = 128                                  # query heads per KV head of a kernel tile


def device_of(device) -> torch.device:
    """``device`` with an index (the current one when it names none)."""
    device = torch.device(device)
    if device.type != "cuda":
        raise _lib.KVQError("kvq kernels run on the GPU only; there is no CPU path")
    return device if device.index is not None else torch.device("cuda", torch.cuda.current_device())


class PromptPlan:
    """The work of an attention over packed sequences of ``lens`` new tokens each, in front of the last of
    ``lens_k`` keys (as many as the new tokens when not given).  Causal: query t of a sequence sees keys
    0 .. t + len_k - len; one that sees none gets zeros.  For ``Hq`` query heads over ``Hkv`` KV heads.  A plan that is dropped is
    kept until the streams of its calls are done with it; it has to live as long as a graph captured with it is replayed."""

    def __init__(self, lens: Sequence[int], Hq: int, Hkv: int, *, lens_k: Optional[Sequence[int]] = None,
                 causal: bool = True, device="cuda"):
        lq = np.ascontiguousarray(lens, dtype=np.int64).reshape(-1)
        lk = lq if lens_k is None else np.ascontiguousarray(lens_k, dtype=np.int64).reshape(-1)
        if lq.shape != lk.shape:
            raise ValueError("lens and lens_k must name the same sequences")
        if (lq < 0).any() or (lk < 0).any():
            raise ValueError("lengths must not be negative")
        if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > MAX_REP:
            raise ValueError(f"{Hq} query heads over {Hkv} KV heads: the quotient must be whole and at most {MAX_REP}")
        if int(lq.sum()) >= 1 << 31 or int(lk.sum()) >= 1 << 31:
            raise ValueError("too many rows")
        self.Hq, self.Hkv, self.causal = int(Hq), int(Hkv), bool(causal)
        self.rows, self.keys = int(lq.sum()), int(lk.sum())
        self.device = device_of(device)
        info = np.zeros(3, dtype=np.int64)
        args = (lq.ctypes.data, lk.ctypes.data, len(lq), self.Hq // self.Hkv, self.Hkv, int(self.causal))
        _lib.call("kvq_prompt_plan", *args, None, 0, info.ctypes.data)
        words = np.empty(max(8 * info[0] + 4 * info[1], 1), dtype=np.int32)
        _lib.call("kvq_prompt_plan", *args, words.ctypes.data, words.size, info.ctypes.data)
        self.items, self.merges, self.parts = info.tolist()
        self.words = torch.from_numpy(words).to(self.device)
        self._streams = {_lib.stream_of(self.words)}     # that the words belong to, or are recorded for

    def workspace_floats(self, d: int) -> int:
        """Float32 scratch of a call at head_dim ``d``: none where the rows fill the chip without cutting along the keys."""
        return _lib.load().kvq_prompt_workspace(self.parts, self.Hkv, d)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float, plan: PromptPlan, *,
                     out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the packed rows q (rows, Hq, d) over k, v (keys, Hkv, d), bf16 or fp16 of one type, head_dim 64
    or 128, any row and head strides of whole 16 bytes (others are copied); returns (rows, Hq, d).  Forward only, as the
    decodes: no gradient is recorded."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks:
        raise ValueError(f"prompt_attention takes q (rows, Hq, d) and k, v (keys, Hkv, d), got {tuple(qs)}, "
                         f"{tuple(ks)}, {tuple(v.shape)}")
    d, dtype = qs[2], q.dtype
    if qs[0] != plan.rows or qs[1] != plan.Hq or ks != (plan.keys, plan.Hkv, d):
        raise ValueError(f"prompt_attention: q {tuple(qs)} and k {tuple(ks)} do not match the plan "
                         f"({plan.rows} rows of {plan.Hq} heads, {plan.keys} keys of {plan.Hkv})")
    if dtype not in (torch.bfloat16, torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise TypeError("prompt_attention takes bf16 or fp16 rows of one type")
    if d not in (64, 128):
        raise _lib.KVQError(f"prompt_attention: head_dim must be 64 or 128 (got {d})")
    device, index = plan.device, plan.device.index
    if q.get_device() != index or k.get_device() != index or v.get_device() != index:
        _lib.require_gpu(q, k, v)
        raise ValueError(f"prompt_attention: the plan is for {device}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _lib.out_or_new(out, qs, dtype, device, "prompt_attention")
    if plan.keys == 0:
        return out.zero_()
    (q, qp, qt, qh), (k, kp, kt, kh), (v, vp, vt, vh) = rows16(q), rows16(k), rows16(v)
    ws, floats = None, 0
    if workspace is not None:
        if workspace.dtype != torch.float32 or not workspace.is_contiguous() or workspace.device != device:
            raise ValueError("workspace must be contiguous float32 on the plan's device")
    elif plan.parts:
        workspace = torch.empty((plan.workspace_floats(d),), dtype=torch.float32, device=device)
    if workspace is not None:
        ws, floats = workspace.data_ptr(), workspace.numel()
    stream = _lib.stream_of(q)
    if stream not in plan._streams and not torch.cuda.is_current_stream_capturing():
        plan.words.record_stream(torch.cuda.current_stream(device))
        plan._streams.add(stream)
    _lib.call_on(device, "kvq_prompt_attention", qp, qt, qh, kp, kt, kh, vp, vt, vh,
                 _lib.DTYPE_CODE[dtype], plan.Hq, plan.Hkv, d, float(scaling), plan.words.data_ptr(), plan.items, plan.merges, plan.parts,
                 out.data_ptr(), ws, floats, stream)
    return out


def rows16(x: torch.Tensor):
    """x (rows, heads, d) with its address, row and head strides, or a copy where the kernels cannot read it in 16-byte
    pieces."""
    at = x.data_ptr()
    st, sh, sd = x.stride()
    if sd != 1 or (st | sh) % 8 or at % 16 or not 0 <= st < 1 << 24:
        x = x.detach().clone(memory_format=torch.contiguous_format)
        at, (st, sh, _) = x.data_ptr(), x.stride()
    return x, at, st, sh
