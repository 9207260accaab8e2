"""Rotary positions: both pair layouts, a part of the head, frequency rules for
long contexts, with or without the append into a paged cache.

The engine's own forward (``pse.engine``) keeps its in-place rotate-half
kernel; these entry points serve models whose positions differ from it, and
calls packed over requests of different lengths.
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
      ``fast`` and ``slow`` times, and a factor 0.1 ln(factor) + 1 on sine and
      cosine (``attention_factor`` overrides it).
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
    return out, _number(scaling, "attention_factor", 0.1 * math.log(factor) + 1.0)


class RotaryPlan:
    """A model's rotary positions: frequencies in turns per position on the
    device (fp64, ``rotary_dim / 2`` entries), the pair layout and the factor.
    Build it once per model and device; it holds no state between calls."""

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
        self.turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=self.device)
        self.spec = N.RotarySpec(self.turns.data_ptr(), self.factor, self.head_dim, self.rotary_dim,
                                 int(self.interleaved))


_NO_HEADS = N.HeadView(None, 0, 0, 0)


def head_view(t: torch.Tensor) -> N.HeadView:
    return N.HeadView(t.data_ptr(), t.stride(0), t.stride(1), t.shape[1])


def check_heads(name: str, t: torch.Tensor, head_dim: int, like: torch.Tensor | None = None,
                heads: int | None = None) -> None:
    """[tokens, heads, head_dim], the last axis contiguous, on a GPU; tokens,
    dtype and device as ``like`` has them."""
    if not torch.is_tensor(t) or t.dim() != 3 or t.shape[2] != head_dim:
        raise ValueError(f"{name} must be a [tokens, heads, {head_dim}] tensor, got "
                         f"{tuple(t.shape) if torch.is_tensor(t) else type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU")
    N.dtype_code(t.dtype)
    if t.stride(2) != 1 and t.numel():
        raise ValueError(f"{name}'s last axis must be contiguous")
    if heads is not None and t.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads, got {t.shape[1]}")
    if like is not None and (t.shape[0] != like.shape[0] or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must match q in tokens, dtype and device")


def check_index(name: str, t: torch.Tensor, n: int, device) -> None:
    if not torch.is_tensor(t) or t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != device or \
            not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on {device}")


def _check_out(name: str, out: torch.Tensor, src: torch.Tensor, head_dim: int) -> None:
    check_heads(name, out, head_dim, src, src.shape[1])
    if out.data_ptr() == src.data_ptr() and out.stride() != src.stride() and src.numel():
        raise ValueError(f"{name} overlaps its input with other strides")


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan, *,
           q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Turn q [T, q_heads, head_dim] and k [T, kv_heads, head_dim] (or None) by
    the tokens' ``positions`` (int32 [T]); any token and head strides (views of
    a fused projection included).  Results go to ``q_out`` / ``k_out`` (which
    may be q / k themselves) or to new tensors, and are returned as (q, k)."""
    check_heads("q", q, plan.head_dim)
    check_index("positions", positions, q.shape[0], q.device)
    if plan.device != q.device:
        raise ValueError(f"the plan is on {plan.device}, q on {q.device}")
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _check_out("q_out", q_out, q, plan.head_dim)
    kv, kv_out = _NO_HEADS, _NO_HEADS
    if k is not None:
        check_heads("k", k, plan.head_dim, q)
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        _check_out("k_out", k_out, k, plan.head_dim)
        kv, kv_out = head_view(k), head_view(k_out)
    N.call("pse_rotary", plan.spec, head_view(q), head_view(q_out), kv, kv_out, positions.data_ptr(), q.shape[0],
           N.dtype_code(q.dtype), N.stream_ptr())
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
    check_heads("q", q, plan.head_dim)
    check_heads("k", k, plan.head_dim, q, cache.n_heads)
    check_heads("v", v, plan.head_dim, q, cache.n_heads)
    if cache.head_dim != plan.head_dim or cache.dtype != q.dtype or cache.device != q.device:
        raise ValueError("the cache must match q in head_dim, dtype and device")
    if plan.device != q.device:
        raise ValueError(f"the plan is on {plan.device}, q on {q.device}")
    if not 0 <= layer < cache.n_layers:
        raise ValueError(f"layer {layer} of a cache with {cache.n_layers}")
    T = q.shape[0]
    for name, t in (("positions", positions), ("slots", slots), ("cache_positions", cache_positions)):
        check_index(name, t, T, q.device)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _check_out("q_out", q_out, q, plan.head_dim)
    kv_out = _NO_HEADS
    if k_out is not None:
        _check_out("k_out", k_out, k, plan.head_dim)
        kv_out = head_view(k_out)
    N.call("pse_rotary_append", cache.state, cache.layer(layer), plan.spec, head_view(q), head_view(q_out),
           head_view(k), kv_out, head_view(v), positions.data_ptr(), slots.data_ptr(), cache_positions.data_ptr(), T,
           N.stream_ptr())
    return q_out
