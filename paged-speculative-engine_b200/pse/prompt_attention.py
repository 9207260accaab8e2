"""Causal attention over packed prompts of different lengths (no padding, no
pages): the form in which a batch of admitted prompts leaves the projection.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _native as N
from .rotary import check_heads, head_view


class PackedPrompts:
    """The packing of one batch of prompts: ``lengths`` tokens each, one after
    the other, and the attention's work list for it (built on the host, one
    copy to the device).  One object serves every layer of a forward and any
    number of calls; it is not changed by them, except for ``status``, where a
    kernel leaves an error (``check_status``)."""

    def __init__(self, lengths, q_heads: int, kv_heads: int, device=None) -> None:
        N.load()
        lens = [int(n) for n in lengths]
        if any(n < 0 for n in lens):
            raise ValueError("a prompt's length is negative")
        if q_heads <= 0 or kv_heads <= 0 or q_heads % kv_heads:
            raise ValueError(f"{q_heads} query heads do not divide into {kv_heads} K/V heads")
        self.lengths = lens
        self.tokens = sum(lens)
        if self.tokens >= 1 << 31:
            raise ValueError(f"{self.tokens} packed tokens (at most 2^31 - 1)")
        self.q_heads, self.kv_heads = int(q_heads), int(kv_heads)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.n_cta = torch.cuda.get_device_properties(self.device).multi_processor_count
        host = np.asarray(lens, dtype=np.int32)
        size = ctypes.c_int64(0)
        args = (host.ctypes.data, len(lens), self.q_heads, self.kv_heads, self.n_cta)
        N.call("pse_prompt_plan", *args, None, 0, ctypes.addressof(size))
        plan = np.empty(size.value + 4, dtype=np.int32)
        N.call("pse_prompt_plan", *args, plan.ctypes.data, size.value, ctypes.addressof(size))
        plan[size.value:] = 0  # the status word's place
        self.n_items = (size.value - (self.n_cta + 4) // 4 * 4) // 4
        self.plan = torch.from_numpy(plan).to(self.device)
        self.status = self.plan[size.value:size.value + 1]

    def offsets(self) -> list:
        """First token of each prompt, and the total."""
        out = [0]
        for n in self.lengths:
            out.append(out[-1] + n)
        return out

    def check_status(self) -> None:
        """Synchronise and raise if a kernel gave up a bounded wait."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError(f"prompt attention failed on the device (status {bits})")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prompts: PackedPrompts, *,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every token to its prompt's tokens up to itself.  q [T,
    q_heads, head_dim], k and v [T, kv_heads, head_dim], float32 or bfloat16,
    any token and head strides (views of a fused projection included); T is
    the packing's total.  ``scale`` defaults to 1 / sqrt(head_dim).  Returns
    [T, q_heads, head_dim] (``out`` if given, which must not overlap the
    inputs)."""
    if not torch.is_tensor(q) or q.dim() != 3:
        raise ValueError("q must be a [tokens, heads, head_dim] tensor")
    hd = q.shape[2]
    if not 0 < hd <= 256:
        raise ValueError(f"head_dim must be 1 to 256, got {hd}")
    check_heads("q", q, hd, heads=prompts.q_heads)
    if q.shape[0] != prompts.tokens:
        raise ValueError(f"{q.shape[0]} tokens, but the prompts hold {prompts.tokens}")
    if q.device != prompts.device:
        raise ValueError(f"the prompts are on {prompts.device}, q on {q.device}")
    check_heads("k", k, hd, q, prompts.kv_heads)
    check_heads("v", v, hd, q, prompts.kv_heads)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    check_heads("out", out, hd, q, prompts.q_heads)
    N.call("pse_prompt_attention", head_view(q), head_view(k), head_view(v), head_view(out), q.shape[0], hd,
           N.dtype_code(q.dtype), 1.0 / math.sqrt(hd) if scale is None else float(scale), prompts.plan.data_ptr(),
           prompts.n_cta, prompts.n_items, prompts.status.data_ptr(), N.stream_ptr())
    return out
