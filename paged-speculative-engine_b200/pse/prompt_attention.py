"""Causal attention over packed prompts of different lengths (no padding, no
pages): the form in which a batch of admitted prompts leaves the projection.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _native as N
from .rotary import head_view, new_result, written_view


class PackedPrompts:
    """The packing of one batch of prompts: ``lengths`` tokens each, one after
    the other, and the attention's work list for it (built on the host, one
    copy to the device: 0.1 ms for 24 prompts of up to 1500 tokens, 2.4 ms for
    32 of 8192, 32 + 8 heads).  One object serves every layer of a forward and any
    number of calls, made with its device current; it is not changed by them,
    except for ``status``, where a kernel leaves an error (``check_status``)."""

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
        self.index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        self.device = torch.device("cuda", self.index)
        self.fn = N.fn("pse_prompt_attention")
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
        self._plan_ptr, self._status_ptr = self.plan.data_ptr(), self.status.data_ptr()

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
    inputs), without a gradient.

    bfloat16 with a head_dim of 64 or 128, at most 128 query heads to a K/V
    head, a positive scale, and q, k, v whose base and strides are multiples of
    16 bytes and whose heads and tokens lie apart runs on the tensor cores.
    Anything else runs in fp32 on the CUDA cores, at some 26 TFLOP/s instead
    of 600 to 1200."""
    shape, dtype, dev = getattr(q, "shape", ()), getattr(q, "dtype", None), prompts.index
    stream = N.stream_on(dev)
    hd = shape[2] if len(shape) == 3 else 0
    if not 0 < hd <= 256:
        raise ValueError(f"q must be [tokens, heads, head_dim] with a head_dim of 1 to 256, got {tuple(shape)}")
    T = prompts.tokens
    qv = head_view("q", q, T, prompts.q_heads, hd, dtype, dev)
    kv = head_view("k", k, T, prompts.kv_heads, hd, dtype, dev)
    vv = head_view("v", v, T, prompts.kv_heads, hd, dtype, dev)
    code = N.dtype_code(dtype)
    if out is None:
        out, ov = new_result(q, qv, hd)
    else:
        ov = written_view("out", out, T, prompts.q_heads, hd, dtype, dev)
    rc = prompts.fn(N.views4(*qv, *kv, *vv, *ov), T, hd, code, 1.0 / math.sqrt(hd) if scale is None else float(scale),
                    prompts._plan_ptr, prompts.n_cta, prompts.n_items, prompts._status_ptr, stream)
    if rc:
        raise N.failed("pse_prompt_attention", rc)
    N.launches["pse_prompt_attention"] += 1
    return out
