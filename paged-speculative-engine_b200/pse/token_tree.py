"""Attention of drafted token trees of any shape over the paged cache.

``pse.tree`` drives trees of equal branches through one kernel rule; here each
request brings its own tree: any parents, any number of nodes (none included),
packed over the requests.  Node j of a request stands in the cache at position
context + j, whatever its depth; its rotary position is context + depth.
"""
from __future__ import annotations

import math

import torch

from . import _native as N
from .rotary import head_view, index_ptr, new_result, written_view

MAX_NODES = 4096  # nodes of one request's tree


class TokenTrees:
    """A batch of trees: ``masks`` int64 [nodes, words] (bit m of a node's
    words: it attends to node m of its own tree), ``counts`` the requests' node
    counts (host integers)."""

    def __init__(self, masks: torch.Tensor, counts, depths: torch.Tensor | None = None,
                 offsets: torch.Tensor | None = None) -> None:
        N.load()
        self.counts = [int(n) for n in counts]
        if any(n < 0 for n in self.counts):
            raise ValueError("a tree's node count is negative")
        self.nodes, self.max_nodes = sum(self.counts), max(self.counts, default=0)
        if self.max_nodes > MAX_NODES:
            raise ValueError(f"a tree of {self.max_nodes} nodes (at most {MAX_NODES})")
        if not torch.is_tensor(masks) or masks.dim() != 2 or masks.dtype != torch.int64 or not masks.is_cuda or \
                not masks.is_contiguous() or masks.shape[0] != self.nodes or masks.shape[1] < 1:
            raise ValueError(f"masks must be a contiguous int64 [{self.nodes}, words] tensor on a GPU")
        self.words = masks.shape[1]
        if self.max_nodes > 64 * self.words:
            raise ValueError(f"{self.words} mask words for a tree of {self.max_nodes} nodes")
        self.masks, self.depths, self.device, self.index = masks, depths, masks.device, masks.get_device()
        self.offsets = _offsets(self.counts, self.device) if offsets is None else offsets
        self._offsets_ptr = index_ptr("offsets", self.offsets, len(self.counts) + 1, self.index)
        self.fn = N.fn("pse_token_tree_attention")
        self._masks_ptr = masks.data_ptr()


def _offsets(counts, device) -> torch.Tensor:
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32).to(device, non_blocking=True)


def tree_masks(parents: torch.Tensor, counts) -> TokenTrees:
    """Ancestor masks of packed trees.  ``parents`` int32 [nodes] on the
    device: a node's parent within its tree (a lower index) or -1 for a child
    of the context.  Each node sees itself and its ancestors; ``depths`` int32
    counts the edges above it (0 for a child of the context)."""
    counts = [int(n) for n in counts]
    if any(n < 0 for n in counts):
        raise ValueError("a tree's node count is negative")
    n = sum(counts)
    if not torch.is_tensor(parents) or not parents.is_cuda:
        raise ValueError("parents must be on a GPU")
    stream = N.stream_on(parents.get_device())
    index_ptr("parents", parents, n, parents.get_device())
    words = max(1, (max(counts, default=0) + 63) // 64)
    offsets = _offsets(counts, parents.device)
    masks = torch.empty(n, words, dtype=torch.int64, device=parents.device)
    depths = torch.empty(n, dtype=torch.int32, device=parents.device)
    trees = TokenTrees(masks, counts, depths, offsets)
    N.call("pse_tree_masks", parents.data_ptr(), offsets.data_ptr(), len(counts), n, words, masks.data_ptr(),
           depths.data_ptr(), stream)
    return trees


_workspace_sizes: dict = {}  # head_dim -> bytes


def token_tree_workspace(head_dim: int, device) -> torch.Tensor:
    """A workspace for ``token_tree_attention``, for callers that keep one (its
    contents do not matter).  Calls that may overlap on the GPU need one each."""
    size = _workspace_sizes.get(head_dim)
    if size is None:
        size = _workspace_sizes[head_dim] = N.size_call("pse_token_tree_workspace", head_dim)
    return torch.empty(size, dtype=torch.uint8, device=device)


def token_tree_attention(q: torch.Tensor, cache, layer: int, slots: torch.Tensor, context: torch.Tensor,
                         trees: TokenTrees, *, scale: float | None = None, out: torch.Tensor | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every tree node to its request's ``context`` (int32 [rows]
    tokens in the cache) and to the nodes its mask names.  q [nodes, q_heads,
    head_dim] in the cache's dtype, any token and head strides; ``slots`` int32
    [rows] (``cache.slots_tensor``).  The nodes' K/V must be in the cache, node
    j at position context + j.  ``scale`` defaults to 1 / sqrt(head_dim).
    Returns [nodes, q_heads, head_dim], without a gradient; a node that sees
    nothing gives zeros.

    A bfloat16 cache with a head_dim of 64 or 128 and pages of 16, 32, 64 or 128
    tokens, a positive scale, and q whose base and strides are multiples of 16
    bytes runs on the tensor cores.  Anything else runs in fp32 on the CUDA
    cores, many times slower where there are more than a few nodes."""
    hd, dtype, dev = cache.head_dim, cache.dtype, trees.index
    stream = N.stream_on(dev)
    if cache.device.index != dev:
        raise ValueError("the cache and the trees must be on one device")
    if not 0 <= layer < cache.n_layers:
        raise ValueError(f"layer {layer} of a cache with {cache.n_layers}")
    qv = head_view("q", q, trees.nodes, None, hd, dtype, dev)
    heads, rows = qv[3], len(trees.counts)
    if heads == 0 or heads % cache.n_heads or heads // cache.n_heads > 64 or hd > 256:
        raise ValueError(f"{heads} query heads over {cache.n_heads} K/V heads of {hd}")
    slot, ctx = index_ptr("slots", slots, rows, dev), index_ptr("context", context, rows, dev)
    if out is None:
        out, ov = new_result(q, qv, hd)
    else:
        ov = written_view("out", out, trees.nodes, heads, hd, dtype, dev)
    if workspace is None:
        workspace = token_tree_workspace(hd, q.device)
    elif workspace.dtype is not torch.uint8 or workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on GPU {dev}")
    rc = trees.fn(cache.state, cache.layer(layer), N.views2(*qv, *ov), slot, ctx, trees._offsets_ptr, rows, trees.nodes,
                  trees.max_nodes, trees._masks_ptr, trees.words, 1.0 / math.sqrt(hd) if scale is None else float(scale),
                  workspace.data_ptr(), workspace.numel(), stream)
    if rc:
        raise N.failed("pse_token_tree_attention", rc)
    N.launches["pse_token_tree_attention"] += 2
    return out
