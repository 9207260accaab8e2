"""Rotary positions: both pair layouts, a part of the head, frequency rules for
long contexts, with or without the append into a paged cache.

The engine's own forward (``pse.engine``) keeps its in-place rotate-half
kernel; these entry points serve models whose positions differ from it, and
calls packed over requests of different lengths.  They serve: results carry no
gradient, whatever the inputs require.
"""
from __future__ import annotations

import math

import torch

from . import _native as N

SCALING_TYPES = ("linear", "ntk", "bands", "yarn")


def _number(scaling: dict, key: str, default=None) -> float:
    x = scaling.get(key, default)
    if not isinstance(x, (int, float)) or isinstance(x, bool) or not math.isfinite(x) or x <= 0:
        raise ValueError(f"scaling needs a positive number {key!r}, got {x!r}")
    return float(x)


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None):
    """The pairs' frequencies (radians per position, Python floats) and the
    factor on sine and cosine.  ``scaling`` is None or a dict with a ``type``:

    * ``linear`` (``factor``): f / factor (positions interpolated).
    * ``ntk`` (``factor``): theta grown to theta * factor^(d / (d - 2)), which
      divides the lowest frequency by the factor and keeps the highest.
    * ``bands`` (``factor``, ``low``, ``high``, ``original``): pairs that turn
      fewer than ``low`` times over the ``original`` length are divided by the
      factor, those that turn more than ``high`` times are kept, the ones
      between blend linearly in their number of turns.
    * ``yarn`` (``factor``, ``original``, ``fast``, ``slow``): the same idea
      with the blend linear in the pair's index, between the indices that turn
      ``fast`` and ``slow`` times, and a factor 0.1 ln(factor) + 1, but at
      least 1, on sine and cosine (``attention_factor`` overrides it).
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    if not (math.isfinite(theta) and theta > 1):
        raise ValueError(f"theta must be a number above 1, got {theta}")
    half = rotary_dim // 2
    f = [theta ** (-2.0 * i / rotary_dim) for i in range(half)]
    if scaling is None:
        return f, 1.0
    kind = scaling.get("type")
    if kind not in SCALING_TYPES:
        raise ValueError(f"scaling type {kind!r} is not one of {SCALING_TYPES}")
    factor = _number(scaling, "factor")
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        base = theta * factor ** (rotary_dim / (rotary_dim - 2))
        return [base ** (-2.0 * i / rotary_dim) for i in range(half)], 1.0
    original = _number(scaling, "original")
    if kind == "bands":
        low, high = _number(scaling, "low"), _number(scaling, "high")
        if not low < high:
            raise ValueError("bands scaling needs low < high")
        out = []
        for x in f:
            turns = original * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append(keep * x + (1.0 - keep) * (x / factor))
        return out, 1.0
    fast, slow = _number(scaling, "fast", 32.0), _number(scaling, "slow", 1.0)
    if not slow < fast:
        raise ValueError("yarn scaling needs slow < fast")

    def index_turning(times: float) -> float:
        return rotary_dim * math.log(original / (2 * math.pi * times)) / (2 * math.log(theta))

    first = max(math.floor(index_turning(fast)), 0)
    last = min(math.ceil(index_turning(slow)), rotary_dim - 1)
    out = []
    for i, x in enumerate(f):
        blend = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
        out.append((1.0 - blend) * x + blend * (x / factor))
    return out, _number(scaling, "attention_factor", 0.1 * math.log(max(factor, 1.0)) + 1.0)


class RotaryPlan:
    """A model's rotary positions: frequencies in turns per position on the
    device (fp64, ``rotary_dim / 2`` entries), the pair layout and the factor.
    Build it once per model and device; it holds no state between calls, which
    are made with that device current."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, theta: float = 10000.0,
                 interleaved: bool = False, scaling: dict | None = None, device=None) -> None:
        N.load()
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim <= 0 or head_dim % 2:
            raise ValueError(f"head_dim must be even and positive, got {head_dim}")
        if not 0 <= rotary_dim <= head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} is not within the head's {head_dim}")
        f, self.factor = rotary_frequencies(rotary_dim, float(theta), scaling)
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), rotary_dim, bool(interleaved)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        self.device = torch.device("cuda", self.index)
        self.fn, self.append_fn = N.fn("pse_rotary"), N.fn("pse_rotary_append")
        self.turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=self.device)
        self.spec = N.RotarySpec(self.turns.data_ptr(), self.factor, self.head_dim, self.rotary_dim,
                                 int(self.interleaved))


_NO_HEADS = (0, 0, 0, 0)


def head_view(name: str, t: torch.Tensor, tokens, heads, head_dim: int, dtype, device: int) -> tuple:
    """The library's view of ``t`` (address, strides, heads), which must be [tokens, heads, head_dim] with
    a contiguous last axis, of ``dtype``, on GPU ``device`` (tokens or heads
    None: any)."""
    try:
        T, H, D = t.shape
        s0, s1, s2 = t.stride()
    except (AttributeError, ValueError, TypeError):
        raise ValueError(f"{name} must be a [tokens, heads, {head_dim}] tensor") from None
    if D != head_dim or (tokens is not None and T != tokens) or (heads is not None and H != heads):
        raise ValueError(f"{name} must be [{'tokens' if tokens is None else tokens}, "
                         f"{'heads' if heads is None else heads}, {head_dim}], got {tuple(t.shape)}")
    if t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name} must be {dtype} on GPU {device}, got {t.dtype} on {t.device}")
    if s2 != 1 and T * H * D:
        raise ValueError(f"{name}'s last axis must be contiguous")
    return t.data_ptr(), s0, s1, H


def written_view(name: str, t: torch.Tensor, tokens: int, heads: int, head_dim: int, dtype, device: int) -> tuple:
    """``head_view`` of a tensor that the kernel writes, whose elements must each
    have a place of their own."""
    view = head_view(name, t, tokens, heads, head_dim, dtype, device)
    if not t.is_contiguous():
        reach = head_dim
        for stride, n in sorted(((view[1], tokens), (view[2], heads))):
            if n > 1 and stride < reach and tokens and heads:
                raise ValueError(f"{name} overlaps itself (strides {t.stride()})")
            reach += max(n - 1, 0) * stride
    return view


def index_ptr(name: str, t: torch.Tensor, n: int, device: int) -> int:
    """The address of ``t``, a contiguous int32 tensor of n entries on GPU ``device``."""
    if not torch.is_tensor(t) or t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != n or \
            t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on GPU {device}")
    return t.data_ptr()


def new_result(src: torch.Tensor, view: tuple, head_dim: int):
    """A contiguous result tensor of the shape of ``src`` ([tokens, heads,
    head_dim], checked as ``view``) and the library's view of it."""
    out, heads = torch.empty_like(src, memory_format=torch.contiguous_format), view[3]
    return out, (out.data_ptr(), heads * head_dim, head_dim, heads)


def _out_view(name: str, out: torch.Tensor, src: torch.Tensor, view: tuple, head_dim: int, dtype, device: int):
    v = written_view(name, out, src.shape[0], view[3], head_dim, dtype, device)
    if v[0] == view[0] and v[1:3] != view[1:3] and src.numel():
        raise ValueError(f"{name} overlaps its input with other strides")
    return v


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan, *,
           q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Turn q [T, q_heads, head_dim] and k [T, kv_heads, head_dim] (or None) by
    the tokens' ``positions`` (int32 [T]); any token and head strides (views of
    a fused projection included).  Results go to ``q_out`` / ``k_out`` (which
    may be q / k themselves) or to new tensors, and are returned as (q, k)."""
    hd, dev, dtype = plan.head_dim, plan.index, getattr(q, "dtype", None)
    stream = N.stream_on(dev)
    qv = head_view("q", q, None, None, hd, dtype, dev)
    code, T = N.dtype_code(dtype), q.shape[0]
    pos = index_ptr("positions", positions, T, dev)
    if q_out is None:
        q_out, qo = new_result(q, qv, hd)
    else:
        qo = _out_view("q_out", q_out, q, qv, hd, dtype, dev)
    kv = ko = _NO_HEADS
    if k is not None:
        kv = head_view("k", k, T, None, hd, dtype, dev)
        if k_out is None:
            k_out, ko = new_result(k, kv, hd)
        else:
            ko = _out_view("k_out", k_out, k, kv, hd, dtype, dev)
    rc = plan.fn(plan.spec, N.views4(*qv, *qo, *kv, *ko), pos, T, code, stream)
    if rc:
        raise N.failed("pse_rotary", rc)
    N.launches["pse_rotary"] += 1
    return q_out, k_out


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, plan: RotaryPlan, cache,
                  layer: int, slots: torch.Tensor, cache_positions: torch.Tensor, *,
                  q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> torch.Tensor:
    """``rotary`` of q and k with the append of the turned k and of v into
    ``cache`` (one layer): token t goes to position ``cache_positions[t]`` of
    slot ``slots[t]`` (int32 [T] each; the positions were reserved by the call
    that grew the rows).  ``positions`` are the rotary positions, which differ
    from the cache's for tree nodes.  ``k_out``, if given, receives the turned
    k as well.  Returns the turned q."""
    hd, dev, dtype = plan.head_dim, plan.index, cache.dtype
    stream = N.stream_on(dev)
    if cache.head_dim != hd or cache.device.index != dev:
        raise ValueError("the cache and the plan must match in head_dim and device")
    if not 0 <= layer < cache.n_layers:
        raise ValueError(f"layer {layer} of a cache with {cache.n_layers}")
    qv = head_view("q", q, None, None, hd, dtype, dev)
    T = q.shape[0]
    kv = head_view("k", k, T, cache.n_heads, hd, dtype, dev)
    vv = head_view("v", v, T, cache.n_heads, hd, dtype, dev)
    pos = index_ptr("positions", positions, T, dev)
    slot = index_ptr("slots", slots, T, dev)
    at = index_ptr("cache_positions", cache_positions, T, dev)
    if q_out is None:
        q_out, qo = new_result(q, qv, hd)
    else:
        qo = _out_view("q_out", q_out, q, qv, hd, dtype, dev)
    ko = _NO_HEADS if k_out is None else _out_view("k_out", k_out, k, kv, hd, dtype, dev)
    rc = plan.append_fn(cache.state, cache.layer(layer), plan.spec, N.views5(*qv, *qo, *kv, *ko, *vv), pos, slot, at, T,
                        stream)
    if rc:
        raise N.failed("pse_rotary_append", rc)
    N.launches["pse_rotary_append"] += 1
    return q_out
