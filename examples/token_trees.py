"""Greedy decoding with token trees drafted by lookup, on the operators of
``pse``: packed prompts (``rotary_append`` + ``prompt_attention``), then rounds
that verify one tree per request in one forward (``tree_masks``,
``rotary_append`` at the nodes' depths, ``token_tree_attention``), keep the
accepted path's K/V (``pse_kv_compact``) and drop the rest.

The draft needs no second model: continuations of earlier occurrences of a
request's last tokens are merged into a tree, so the requests' trees differ in
shape and size from round to round (a tree of one node is plain decoding).  The
output is the greedy continuation whatever the trees hold.

    python examples/token_trees.py [--requests 8] [--new-tokens 128] [--nodes 24]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "paged-speculative-engine_b200"))
import pse  # noqa: E402
from pse import _native as N  # noqa: E402


def lookup_tree(history: list, max_nodes: int, depth: int = 8) -> tuple:
    """(tokens, parents) of a tree whose node 0 is the last token of
    ``history`` (sampled, not yet in the cache) and whose paths continue it the
    way earlier occurrences of the same ending went on, the latest first."""
    tokens, parents, children = [history[-1]], [-1], {}
    for n in (3, 2, 1):
        tail = history[-n:]
        for at in range(len(history) - n - 1, -1, -1):
            if len(tokens) >= max_nodes:
                return tokens, parents
            if history[at:at + n] != tail:
                continue
            node = 0
            for token in history[at + n:at + n + depth]:
                child = children.get((node, token))
                if child is None:
                    if len(tokens) >= max_nodes:
                        break
                    child = children[node, token] = len(tokens)
                    tokens.append(token)
                    parents.append(node)
                node = child
    return tokens, parents


class TreeDecoder:
    """Greedy decoding of a batch with a ``pse.TinyLlama`` on the GPU."""

    def __init__(self, model: pse.TinyLlama, *, block_size: int = 16, num_blocks: int = 4096) -> None:
        cfg, w = model.cfg, model.token_emb.weight
        self.model, self.cfg, self.device = model, cfg, w.device
        self.hd = cfg.d_model // cfg.n_heads
        self.cache = pse.PagedKVCache(cfg.n_layers, cfg.n_kv_heads, self.hd, block_size, num_blocks, dtype=w.dtype,
                                      device=w.device)
        self.plan = pse.RotaryPlan(self.hd, theta=cfg.rope_theta, device=w.device)
        self.workspace = pse.token_tree.token_tree_workspace(self.hd, w.device)
        self.rows: dict = {}  # request id -> tokens so far, the last one not in the cache
        self.calls = 0

    def _i32(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device, non_blocking=True)

    def _forward(self, ids, positions, slots, cache_positions, attention) -> torch.Tensor:
        """The model over packed tokens; ``attention(layer, q, k, v)`` is the rows' attention."""
        cfg, hd = self.cfg, self.hd
        x = self.model.token_emb(ids)
        for i, block in enumerate(self.model.blocks):
            h = F.rms_norm(x, (cfg.d_model,), block.norm1.weight, cfg.norm_eps)
            qkv = block.attn.qkv(h).view(len(ids), -1, hd)  # the heads are views of one projection
            q, k, v = qkv.split([cfg.n_heads, cfg.n_kv_heads, cfg.n_kv_heads], 1)
            turned_k = torch.empty_like(k, memory_format=torch.contiguous_format)
            q = pse.rotary_append(q, k, v, positions, self.plan, self.cache, i, slots, cache_positions, k_out=turned_k)
            x = x + block.attn.out(attention(i, q, turned_k, v).flatten(1))
            gate, up = block.gate_up(F.rms_norm(x, (cfg.d_model,), block.norm2.weight, cfg.norm_eps)).chunk(2, -1)
            x = x + block.down(F.silu(gate) * up)
        self.calls += 1
        return self.model.lm_head(F.rms_norm(x, (cfg.d_model,), self.model.norm_f.weight, cfg.norm_eps))

    def _reserve(self, names, widths) -> torch.Tensor:
        """Grow the rows (lengths on the host and the device); their slots."""
        cache = self.cache
        longest = [cache.length(n) + w for n, w in zip(names, widths)]
        cache.ensure_capacity_len(max(longest))
        slots, wide = cache.slots_tensor(names), self._i32(widths)
        base = torch.empty_like(slots)
        N.call("pse_kv_reserve_rows", cache.state, slots.data_ptr(), len(names), wide.data_ptr(), base.data_ptr(),
               N.stream_ptr())
        cache.note_lengths(names, longest)
        return slots

    @torch.no_grad()
    def prefill(self, prompts: dict) -> None:
        """Admit prompts (request id -> tokens) in one packed forward; each
        request's first new token follows from it."""
        names, lengths = list(prompts), [len(p) for p in prompts.values()]
        if not names or min(lengths) == 0:
            raise ValueError("a prompt needs at least one token")
        for n in names:
            self.cache.create_request(n)
        slots = self._reserve(names, lengths)
        ids = self._i32([t for p in prompts.values() for t in p])
        at = self._i32([i for n in lengths for i in range(n)])
        token_slots = slots.repeat_interleave(self._i32(lengths))
        packing = pse.PackedPrompts(lengths, self.cfg.n_heads, self.cfg.n_kv_heads, device=self.device)
        logits = self._forward(ids, at, token_slots, at,
                               lambda layer, q, k, v: pse.prompt_attention(q, k, v, packing))
        last = torch.tensor(packing.offsets()[1:], device=self.device) - 1
        first = logits[last].argmax(-1).tolist()
        packing.check_status()
        self.cache.check_status("prefill")
        for n, t in zip(names, first):
            self.rows[n] = list(prompts[n]) + [t]

    @torch.no_grad()
    def round(self, names, max_nodes: int) -> None:
        """Draft, verify and accept one tree per request."""
        cache = self.cache
        drafts = [lookup_tree(self.rows[n], max_nodes) for n in names]
        counts, context = [len(t) for t, _ in drafts], [cache.length(n) for n in names]
        trees = pse.tree_masks(self._i32([p for _, parents in drafts for p in parents]), counts)
        slots, ctx = self._reserve(names, counts), self._i32(context)
        reps = self._i32(counts)
        start = ctx.repeat_interleave(reps)
        # a node stands at context + its index, and turns by context + its depth
        at = self._i32([c + j for c, n in zip(context, counts) for j in range(n)])
        logits = self._forward(
            self._i32([t for tokens, _ in drafts for t in tokens]), start + trees.depths, slots.repeat_interleave(reps),
            at, lambda layer, q, k, v: pse.token_tree_attention(q, cache, layer, slots, ctx, trees,
                                                                workspace=self.workspace))
        after = logits.argmax(-1).tolist()
        cache.check_status("the tree's verification")

        first, paths = 0, []
        for n, (tokens, parents), count in zip(names, drafts, counts):
            children = {(p, t): j for j, (p, t) in enumerate(zip(parents, tokens)) if j}
            path, node = [], 0
            while node is not None:
                path.append(node)
                self.rows[n].append(after[first + node])
                node = children.get((node, after[first + node]))
            paths.append(path)
            first += count
        # the path's K/V moves up behind the context, the rest is dropped
        longest, st = max(len(p) for p in paths), N.stream_ptr()
        src = self._i32([p + [0] * (longest - len(p)) for p in paths])
        kept, new = self._i32([len(p) for p in paths]), [c + len(p) for c, p in zip(context, paths)]
        for layer in range(cache.n_layers):
            N.call("pse_kv_compact", cache.state, cache.layer(layer), slots.data_ptr(), ctx.data_ptr(), src.data_ptr(),
                   kept.data_ptr(), len(names), longest, st)
        lengths = self._i32(new)
        N.call("pse_kv_truncate", cache.state, slots.data_ptr(), len(names), lengths.data_ptr(), None, None, st)
        cache.note_lengths(names, new)

    def generate(self, prompts: dict, new_tokens: int, max_nodes: int) -> dict:
        """The greedy continuations: request id -> ``new_tokens`` tokens."""
        self.prefill(prompts)
        while True:
            live = [n for n in prompts if len(self.rows[n]) < len(prompts[n]) + new_tokens]
            if not live:
                break
            self.round(live, max_nodes)
        out = {n: self.rows.pop(n)[len(p):len(p) + new_tokens] for n, p in prompts.items()}
        self.cache.free_requests(list(prompts))
        return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--new-tokens", type=int, default=128)
    ap.add_argument("--nodes", type=int, default=24, help="most nodes of a request's tree")
    ap.add_argument("--dtype", choices=("bf16", "f32"), default="bf16")
    args = ap.parse_args()
    torch.manual_seed(0)
    cfg = pse.LlamaConfig(vocab_size=512, d_model=1024, n_layers=4, n_heads=16, n_kv_heads=4, d_ff=2048)
    model = pse.TinyLlama(cfg).to("cuda", torch.bfloat16 if args.dtype == "bf16" else torch.float32)
    g = torch.Generator().manual_seed(1)
    prompts = {f"r{i}": torch.randint(0, cfg.vocab_size, (17 + 37 * i,), generator=g).tolist()
               for i in range(args.requests)}
    for nodes in (1, args.nodes):
        dec = TreeDecoder(model)
        dec.generate(prompts, 4, nodes)
        dec.calls = 0
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = dec.generate(prompts, args.new_tokens, nodes)
        t = time.perf_counter() - t
        n = sum(len(x) for x in out.values())
        print(f"trees of at most {nodes:3d} nodes: {n} tokens in {dec.calls} forwards, {t * 1e3:.0f} ms")


if __name__ == "__main__":
    main()
