"""The token-tree example: its continuations are the greedy ones, whatever the
trees hold.  Against a dense forward in 64 bits; the fp32 forward's logits
differ from it by some 1e-5, and a position whose two best logits are closer
than 1e-3 ends the comparison of its request (none does in these cases unless a
weight changes).  GPU only."""
from __future__ import annotations

import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def dense_logits(model, ids):
    """fp64 logits of every position."""
    cfg = model.cfg
    hd, T = cfg.d_model // cfg.n_heads, len(ids)
    w = {n: p.detach().double() for n, p in model.named_parameters()}

    def norm(x, weight):
        return x / (x.pow(2).mean(-1, keepdim=True) + cfg.norm_eps).sqrt() * weight

    pos = torch.arange(T, dtype=torch.float64, device="cuda")
    angle = pos[:, None] * cfg.rope_theta ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turn(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    x = w["token_emb.weight"][torch.tensor(ids, device="cuda")]
    hidden = torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1)
    for i in range(cfg.n_layers):
        p = f"blocks.{i}."
        qkv = (norm(x, w[p + "norm1.weight"]) @ w[p + "attn.qkv.weight"].T).view(T, -1, hd)
        q, k, v = qkv.split([cfg.n_heads, cfg.n_kv_heads, cfg.n_kv_heads], 1)
        group = cfg.n_heads // cfg.n_kv_heads
        k, v = turn(k).repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("qhd,khd->hqk", turn(q), k) / math.sqrt(hd)
        o = torch.einsum("hqk,khd->qhd", s.masked_fill(hidden, -math.inf).softmax(-1), v)
        x = x + o.reshape(T, -1) @ w[p + "attn.out.weight"].T
        gate, up = (norm(x, w[p + "norm2.weight"]) @ w[p + "gate_up.weight"].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w[p + "down.weight"].T
    return norm(x, w["norm_f.weight"]) @ w["lm_head.weight"].T


def test_lookup_tree_is_a_tree():
    import token_trees
    tokens, parents = token_trees.lookup_tree([1, 2, 3, 1, 2, 4, 1, 2], 6)
    assert tokens[0] == 2 and parents[0] == -1
    assert all(0 <= p < i for i, p in enumerate(parents) if i)
    assert len(set(zip(parents, tokens))) == len(tokens) <= 6
    assert {t for p, t in zip(parents, tokens) if p == 0} == {3, 4}
    assert token_trees.lookup_tree([7], 6) == ([7], [-1])
    assert token_trees.lookup_tree([7, 7, 7], 1) == ([7], [-1])


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,nodes,bs", [(4, 2, 24, 16), (4, 4, 5, 4), (8, 1, 70, 32), (4, 2, 1, 16)])
def test_trees_decode_greedily(heads, kv_heads, nodes, bs):
    import pse
    import token_trees
    torch.manual_seed(heads + nodes)
    cfg = pse.LlamaConfig(vocab_size=48, d_model=64 * heads, n_layers=2, n_heads=heads, n_kv_heads=kv_heads, d_ff=192)
    model = pse.TinyLlama(cfg).cuda()
    g = torch.Generator().manual_seed(3)
    prompts = {n: torch.randint(0, 12, (length,), generator=g).tolist()
               for n, length in (("a", 1), ("b", 40), ("c", 129), ("d", 17))}
    dec = token_trees.TreeDecoder(model, block_size=bs, num_blocks=4096 // bs)
    out = dec.generate(prompts, 40, nodes)
    assert dec.cache.allocator.num_free == 4096 // bs
    assert dec.calls <= 40 if nodes > 1 else dec.calls == 40
    compared = 0
    for n, prompt in prompts.items():
        assert len(out[n]) == 40
        logits = dense_logits(model, prompt + out[n])[len(prompt) - 1:-1]
        best = logits.topk(2, -1)
        for i, token in enumerate(out[n]):
            if float(best.values[i, 0] - best.values[i, 1]) < 1e-3:
                break
            assert token == int(best.indices[i, 0]), (n, i)
            compared += 1
    assert compared >= 100


@pytest.mark.gpu
def test_trees_save_forwards():
    """A history that repeats is drafted right: fewer forwards than tokens."""
    import pse
    import token_trees
    torch.manual_seed(0)
    cfg = pse.LlamaConfig(vocab_size=16, d_model=128, n_layers=1, n_heads=2, n_kv_heads=2, d_ff=64)
    dec = token_trees.TreeDecoder(pse.TinyLlama(cfg).to("cuda", torch.bfloat16))
    out = dec.generate({"r": [1, 2, 3]}, 200, 16)
    assert len(out["r"]) == 200 and dec.calls < 200
