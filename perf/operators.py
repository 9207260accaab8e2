"""Cases and plain forms of the operators a request passes through around its
paged KV cache: rotary positions (with the append into the cache's pages),
attention over packed prompts, and attention of drafted token trees over the
cache.

``own`` False computes every operator from elementary torch operations in 32
bits; True makes the calls a user of ``pse`` makes.  ``exact`` states the
definitions once more in 64 bits.

Definitions (all shapes packed over tokens or tree nodes, heads grouped: query
head h reads K/V head h // (q_heads / kv_heads)):

* rotary: pair i of the first ``rotary_dim`` elements of a head turns by the
  angle position * f_i; pairs are (i, i + rotary_dim/2) ("half") or (2i, 2i+1)
  ("interleaved"); f_i = theta^(-2i/rotary_dim), rescaled for long contexts by
  one of the rules of ``_frequencies``; the rest of the head passes through.
* rotary_append: the same, with the turned K and the V written to their
  tokens' places in the cache's pages.
* prompt attention: token i of a prompt attends to tokens 0..i of that prompt.
* tree attention: node n of a request attends to the request's whole context
  (in the cache) and to the nodes its mask names (its ancestors and itself),
  whose K/V stand in the cache after the context.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 8.0},
    "bands": {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"type": "yarn", "factor": 16.0, "fast": 32.0, "slow": 1.0, "original": 8192},
}


def _pse():
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "paged-speculative-engine_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import pse
    return pse


# ---------------------------------------------------------------- cases
def _rotary(name, tokens, heads, head_dim, rotary_dim, layout, scaling, max_position, dtype):
    return {"name": name, "op": "rotary", "tokens": tokens, "q_heads": heads[0], "kv_heads": heads[1],
            "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": layout == "interleaved", "scaling": scaling,
            "max_position": max_position, "dtype": dtype}


def _append(name, requests, shortest, longest, spread, heads, head_dim, rotary_dim, layout, scaling, block, dtype):
    return {"name": name, "op": "rotary_append", "requests": requests, "shortest": shortest, "longest": longest,
            "spread": spread, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": head_dim,
            "rotary_dim": rotary_dim, "interleaved": layout == "interleaved", "scaling": scaling,
            "block_size": block, "dtype": dtype}


def _prompt(name, prompts, shortest, longest, spread, heads, head_dim, dtype):
    return {"name": name, "op": "prompt", "prompts": prompts, "shortest": shortest, "longest": longest,
            "spread": spread, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": head_dim, "dtype": dtype}


def _tree(name, requests, shortest, longest, fewest, most, spread, heads, head_dim, block, dtype):
    return {"name": name, "op": "tree", "requests": requests, "shortest": shortest, "longest": longest,
            "fewest": fewest, "most": most, "spread": spread, "q_heads": heads[0], "kv_heads": heads[1],
            "head_dim": head_dim, "block_size": block, "dtype": dtype}


def listed():
    return [
        # one decode step's tokens of the Llama-style pair: a call of a few microseconds
        _rotary("rotary-decode", 48, (32, 8), 64, 64, "half", "none", 16384, "bf16"),
        # a whole prefill batch with positions far past the trained length
        _rotary("rotary-prompt", 16384, (32, 8), 128, 128, "half", "bands", 131072, "bf16"),
        # the fp32 engine; neighbouring pairs, a part of an odd head size, an odd count
        _rotary("rotary-partial-f32", 5003, (16, 16), 80, 32, "interleaved", "yarn", 65536, "f32"),
        # prompts of different lengths entering the cache
        _append("append-prompts", 24, 17, 1500, 1, (32, 8), 64, 64, "half", "none", 32, "bf16"),
        # one short prompt: latency
        _prompt("prompt-short", 1, 37, 37, 2, (12, 12), 64, "bf16"),
        # an admission round of the Llama-style pair: ragged prompts, grouped heads
        _prompt("prompt-mixed", 24, 17, 1500, 3, (32, 8), 64, "bf16"),
        # long documents, wide heads: bound by the tensor cores
        _prompt("prompt-long", 3, 5003, 8192, 4, (32, 8), 128, "bf16"),
        # the fp32 engine's prompts
        _prompt("prompt-f32", 5, 8, 300, 5, (12, 12), 64, "f32"),
        # one request, a small tree: latency
        _tree("tree-short", 1, 300, 300, 8, 8, 6, (12, 12), 64, 16, "bf16"),
        # a serving batch of ragged contexts and trees
        _tree("tree-batch", 64, 128, 4096, 5, 26, 7, (32, 8), 64, 16, "bf16"),
        # long contexts, large trees: the cache's bytes and the tensor cores both count
        _tree("tree-long", 12, 8001, 32768, 60, 64, 8, (32, 8), 128, 64, "bf16"),
        # the fp32 engine's cache
        _tree("tree-f32", 8, 17, 1000, 1, 12, 9, (12, 12), 64, 16, "f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_once(rng):
    heads = rng.choice([(12, 12), (32, 8), (16, 4), (6, 6), (16, 2), (24, 3), (10, 2)])
    head_dim = rng.choice([64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    spread = rng.randrange(1000, 1 << 30)
    layout = rng.choice(["half", "interleaved"])
    scaling = rng.choice(sorted(_SCALINGS))
    rotary_dim = max(16, int(head_dim * rng.choice([1, 1, 0.5, 0.25])))
    block = rng.choice([16, 32, 64])
    op = rng.choice(["rotary", "rotary_append", "prompt", "tree"])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, head_dim])
        rotary_dim = rng.choice([head_dim, head_dim // 2, 32])
        return _rotary("", _log_int(rng, 1, 16384), heads, head_dim, rotary_dim, layout, scaling,
                       _log_int(rng, 4096, 131072), dtype)
    if op == "rotary_append":
        longest = _log_int(rng, 8, 2000)
        return _append("", _log_int(rng, 1, 64), _log_int(rng, 1, longest), longest, spread, heads, head_dim,
                       rotary_dim, layout, scaling, block, dtype)
    if op == "prompt":
        longest = _log_int(rng, 8, 8192 if dtype == "bf16" else 1024)
        return _prompt("", _log_int(rng, 1, 32), _log_int(rng, 1, longest), longest, spread, heads, head_dim, dtype)
    longest = _log_int(rng, 32, 32768 if dtype == "bf16" else 4096)
    most = _log_int(rng, 1, 64)
    return _tree("", _log_int(rng, 1, 96), _log_int(rng, 1, longest), longest, _log_int(rng, 1, most), most, spread,
                 heads, head_dim, block, dtype)


def draw(rng):
    ceiling = {}
    for c in listed():
        w = work(c)
        for key in (c["op"], (c["op"], c["dtype"])):
            b, f = ceiling.get(key, (0, 0))
            ceiling[key] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        case = _draw_once(rng)
        w = work(case)
        # an fp32 attention call is held to a sixteenth of the largest bf16 one
        b, f = ceiling[case["op"]]
        part = 16 if case["dtype"] == "f32" and case["op"] in ("prompt", "tree") else 1
        if w["bytes"] <= b / part and w["flops"] <= f / part:
            del case["name"]
            return case


def _spread_sizes(n, lo, hi, spread):
    """n whole numbers over [lo, hi], even over their logarithm; the largest is hi."""
    rng = random.Random(spread)
    sizes = [_log_int(rng, lo, hi) for _ in range(n)]
    sizes[rng.randrange(n)] = hi
    return sizes


def _lengths(case):
    n = case["prompts"] if case["op"] == "prompt" else case["requests"]
    return _spread_sizes(n, case["shortest"], case["longest"], case["spread"])


def _node_counts(case):
    return _spread_sizes(case["requests"], case["fewest"], case["most"], case["spread"] + 1)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    hq, hk, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        t = case["tokens"]
        return {"bytes": 2 * t * (hq + hk) * hd * size + 4 * t, "flops": 3 * t * (hq + hk) * case["rotary_dim"]}
    if case["op"] == "rotary_append":
        t = sum(_lengths(case))
        # q, k, v in; q, the cache's k and v, and the packed k out
        return {"bytes": t * (2 * hq + 5 * hk) * hd * size + 12 * t, "flops": 3 * t * (hq + hk) * case["rotary_dim"]}
    if case["op"] == "prompt":
        lens = _lengths(case)
        return {"bytes": sum(lens) * (2 * hq + 2 * hk) * hd * size,
                "flops": 4 * hq * hd * sum(n * (n + 1) // 2 for n in lens)}
    ctx, nodes = _lengths(case), _node_counts(case)
    return {"bytes": sum((c + n) * 2 * hk * hd * size + n * 2 * hq * hd * size for c, n in zip(ctx, nodes)),
            "flops": 4 * hq * hd * sum(n * (c + 1) for c, n in zip(ctx, nodes))}


# ---------------------------------------------------------------- inputs
def _frequencies(rotary_dim, scaling, theta=10000.0):
    """f_i (radians per position) in double precision, and the factor on both
    sine and cosine.  linear: f / factor.  ntk: theta grows so that the lowest
    frequency is divided by the factor.  bands: wavelengths longer than
    original / low are divided by the factor, those shorter than original /
    high are kept, with a linear blend between.  yarn: the same blend over the
    pair's index, between the indices whose pairs turn `fast` and `slow` times
    over the original length, with a temperature on the logits."""
    f = [theta ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    s = _SCALINGS[scaling]
    if s is None:
        return f, 1.0
    if s["type"] == "linear":
        return [x / s["factor"] for x in f], 1.0
    if s["type"] == "ntk":
        base = theta * s["factor"] ** (rotary_dim / (rotary_dim - 2))
        return [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)], 1.0
    if s["type"] == "bands":
        out = []
        for x in f:
            keep = (s["original"] * x / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])
            keep = min(1.0, max(0.0, keep))
            out.append(keep * x + (1 - keep) * x / s["factor"])
        return out, 1.0
    index = [rotary_dim * math.log(s["original"] / (t * 2 * math.pi)) / (2 * math.log(theta))
             for t in (s["fast"], s["slow"])]
    lo, hi = max(0, math.floor(index[0])), min(rotary_dim - 1, math.ceil(index[1]))
    out = []
    for i, x in enumerate(f):
        blend = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
        out.append(blend * x / s["factor"] + (1 - blend) * x)
    return out, 0.1 * math.log(s["factor"]) + 1.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda").to(_DTYPES[dtype])


def _fused(case, tokens, gen):
    """q, k, v as views of one fused projection's rows, as a model's forward has them."""
    hq, hk, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    rows = _normal(gen, case["dtype"], tokens, (hq + 2 * hk) * hd)
    heads = rows.view(tokens, hq + 2 * hk, hd)
    return heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:]


def _tables(lengths, block, chunks=3):
    """Block tables after the requests' tokens entered the cache a third at a
    time, request after request, blocks taken from the end of the free list;
    and the order of those steps as (request, first, count)."""
    total = sum((n + block - 1) // block for n in lengths)
    free, tables, steps = list(range(total)), [[] for _ in lengths], []
    done = [0] * len(lengths)
    for c in range(chunks):
        for r, n in enumerate(lengths):
            upto = n * (c + 1) // chunks
            if upto > done[r]:
                steps.append((r, done[r], upto - done[r]))
                done[r] = upto
                while len(tables[r]) * block < upto:
                    tables[r].append(free.pop())
    return total, tables, steps


def _offsets(sizes):
    out = [0]
    for n in sizes:
        out.append(out[-1] + n)
    return out


def _inputs(case, seed):
    gen = _gen(seed)
    if case["op"] == "rotary":
        q, k, _ = _fused(case, case["tokens"], gen)
        pos = torch.randint(0, case["max_position"], (case["tokens"],), generator=gen, device="cuda", dtype=torch.int32)
        return {"q": q, "k": k, "positions": pos}
    if case["op"] == "rotary_append":
        lens = _lengths(case)
        q, k, v = _fused(case, sum(lens), gen)
        pos = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in lens])
        return {"q": q, "k": k, "v": v, "positions": pos, "lengths": lens}
    if case["op"] == "prompt":
        lens = _lengths(case)
        q, k, v = _fused(case, sum(lens), gen)
        return {"q": q, "k": k, "v": v, "lengths": lens}
    ctx, nodes = _lengths(case), _node_counts(case)
    # each request's context, then its tree's nodes
    every = [c + n for c, n in zip(ctx, nodes)]
    k = _normal(gen, case["dtype"], sum(every), case["kv_heads"], case["head_dim"])
    v = _normal(gen, case["dtype"], sum(every), case["kv_heads"], case["head_dim"])
    q = _fused(case, sum(nodes), gen)[0]
    rng = random.Random(seed)
    words = (max(nodes) + 63) // 64
    masks = torch.zeros(sum(nodes), words * 64, dtype=torch.bool)
    first = 0
    for n in nodes:
        for i in range(n):
            parent = rng.randrange(-1, i) if i < 4 else rng.randrange(i // 2, i)
            if parent >= 0:
                masks[first + i] = masks[first + parent]
            masks[first + i, i] = True
        first += n
    return {"q": q, "k": k, "v": v, "context": ctx, "nodes": nodes, "visible": masks}


def _words(visible):
    """[n, 64 w] truth values as [n, w] int64 words, bit b of word w for node 64 w + b."""
    bits = visible.view(visible.shape[0], -1, 64).to(torch.int64)
    return (bits << torch.arange(64)).sum(-1)


def _pools(case, k, v, lengths):
    """The cache's pages holding packed k, v (as _tables places them)."""
    block = case["block_size"]
    total, tables, _ = _tables(lengths, block)
    off = _offsets(lengths)
    pools = []
    for x in (k, v):
        pool = torch.zeros(total, case["kv_heads"], block, case["head_dim"], dtype=x.dtype, device="cuda")
        for r, n in enumerate(lengths):
            b, p = _places(tables[r], n, block)
            pool[b, :, p] = x[off[r]:off[r + 1]]
        pools.append(pool)
    return pools[0], pools[1], tables


def _places(table, n, block):
    at = torch.arange(n, device="cuda")
    return torch.tensor(table, device="cuda")[at // block], at % block


def _cache(case, k, v, lengths):
    """A pse cache holding packed k, v, filled through its public calls."""
    block = case["block_size"]
    total, tables, steps = _tables(lengths, block)
    cache = _pse().PagedKVCache(1, case["kv_heads"], case["head_dim"], block, total, dtype=_DTYPES[case["dtype"]],
                                max_requests=len(lengths), max_blocks_per_request=max(len(t) for t in tables))
    off = _offsets(lengths)
    ids = ["r%d" % r for r in range(len(lengths))]
    for r in ids:
        cache.create_request(r)
    for r, first, n in steps:
        at = slice(off[r] + first, off[r] + first + n)
        cache.append(ids[r], [k[at].transpose(0, 1)], [v[at].transpose(0, 1)])
    return cache, cache.slots_tensor(ids)


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    op = case["op"]
    if op in ("rotary", "rotary_append"):
        if own:
            st["plan"] = _pse().RotaryPlan(case["head_dim"], rotary_dim=case["rotary_dim"],
                                           interleaved=case["interleaved"], scaling=_SCALINGS[case["scaling"]])
        else:
            f, st["factor"] = _frequencies(case["rotary_dim"], case["scaling"])
            st["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if op == "rotary_append":
        zero = torch.zeros_like(st["k"])
        if own:
            st["cache"], slots = _cache(case, zero, zero, st["lengths"])
            st["slots"] = slots.repeat_interleave(torch.tensor(st["lengths"], device="cuda"))
        else:
            st["k_pool"], st["v_pool"], tables = _pools(case, zero, zero, st["lengths"])
            places = [_places(t, n, case["block_size"]) for t, n in zip(tables, st["lengths"])]
            st["block"], st["row"] = torch.cat([p[0] for p in places]), torch.cat([p[1] for p in places])
    if op == "prompt" and own:
        st["prompts"] = _pse().PackedPrompts(st["lengths"], case["q_heads"], case["kv_heads"])
    if op == "tree":
        st["masks"] = _words(st["visible"]).cuda()
        st["visible"] = st["visible"].cuda()
        every = [c + n for c, n in zip(st["context"], st["nodes"])]
        if own:
            st["cache"], st["slots"] = _cache(case, st["k"], st["v"], every)
            st["context"] = torch.tensor(st["context"], dtype=torch.int32, device="cuda")
            st["trees"] = _pse().TokenTrees(st["masks"], st["nodes"])
        else:
            st["k_pool"], st["v_pool"], tables = _pools(case, st["k"], st["v"], every)
            st["tables"] = [torch.tensor(t, device="cuda") for t in tables]
        del st["k"], st["v"]
    return st


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        pse = _pse()
        if op == "rotary":
            return pse.rotary(state["q"], state["k"], state["positions"], state["plan"])
        if op == "rotary_append":
            cache = state["cache"]
            k_out = torch.empty_like(state["k"], memory_format=torch.contiguous_format)
            q = pse.rotary_append(state["q"], state["k"], state["v"], state["positions"], state["plan"], cache, 0,
                                  state["slots"], state["positions"], k_out=k_out)
            return q, k_out, cache.k_pool[0], cache.v_pool[0]
        if op == "prompt":
            return pse.prompt_attention(state["q"], state["k"], state["v"], state["prompts"])
        return pse.token_tree_attention(state["q"], state["cache"], 0, state["slots"], state["context"],
                                        state["trees"])
    if op == "rotary":
        cos, sin = _turns(state)
        return _turned(state["case"], state["q"], cos, sin), _turned(state["case"], state["k"], cos, sin)
    if op == "rotary_append":
        cos, sin = _turns(state)
        q, k = _turned(state["case"], state["q"], cos, sin), _turned(state["case"], state["k"], cos, sin)
        state["k_pool"][state["block"], :, state["row"]] = k
        state["v_pool"][state["block"], :, state["row"]] = state["v"]
        return q, k, state["k_pool"], state["v_pool"]
    return _plain_prompt(state) if op == "prompt" else _plain_tree(state)


def _turns(state):
    # The angle is reduced to one turn in 64 bits: at position 131071 a 32-bit
    # product is off by several thousandths of a radian.  The rest is 32 bits.
    angle = state["positions"].double()[:, None] * state["frequencies"]
    angle = torch.remainder(angle, 2 * math.pi).float()
    return torch.cos(angle) * state["factor"], torch.sin(angle) * state["factor"]


def _turned(case, x, cos, sin):
    rd = case["rotary_dim"]
    cos, sin = cos[:, None], sin[:, None]
    y = x.float()
    if case["interleaved"]:
        a, b = y[..., 0:rd:2], y[..., 1:rd:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., : rd // 2], y[..., rd // 2: rd]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., rd:]), -1).to(x.dtype)


def _softmax_rows(scores, visible):
    """Softmax over the last axis where `visible`; rows that see nothing are zero."""
    scores = torch.where(visible, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_prompt(state):
    case = state["case"]
    group, scale = case["q_heads"] // case["kv_heads"], 1.0 / math.sqrt(case["head_dim"])
    out = torch.empty(state["q"].shape, dtype=state["q"].dtype, device="cuda")
    first = 0
    for n in state["lengths"]:
        at = slice(first, first + n)
        first += n
        visible = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            q = state["q"][at, heads].float().transpose(0, 1)
            k, v = state["k"][at, h].float(), state["v"][at, h].float()
            p = _softmax_rows(torch.matmul(q, k.t()) * scale, visible)
            out[at, heads] = torch.matmul(p, v).transpose(0, 1).to(out.dtype)
    return out


def _plain_tree(state):
    case = state["case"]
    hk, hd = case["kv_heads"], case["head_dim"]
    group, scale = case["q_heads"] // hk, 1.0 / math.sqrt(hd)
    out = torch.empty(state["q"].shape, dtype=state["q"].dtype, device="cuda")
    first = 0
    for table, c, n in zip(state["tables"], state["context"], state["nodes"]):
        at = slice(first, first + n)
        first += n
        k, v = (p[table].transpose(0, 1).reshape(hk, -1, hd)[:, : c + n].float()
                for p in (state["k_pool"], state["v_pool"]))
        q = state["q"][at].float().view(n, hk, group, hd).permute(1, 2, 0, 3).reshape(hk, group * n, hd)
        visible = torch.cat((torch.ones(n, c, dtype=torch.bool, device="cuda"), state["visible"][at, :n]), 1)
        p = _softmax_rows((torch.matmul(q, k.transpose(1, 2)) * scale).view(hk, group, n, c + n), visible)
        o = torch.matmul(p.view(hk, group * n, c + n), v).view(hk, group, n, hd)
        out[at] = o.permute(2, 0, 1, 3).reshape(n, hk * group, hd).to(out.dtype)
    return out


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] in ("rotary", "rotary_append"):
        f, factor = _frequencies(case["rotary_dim"], case["scaling"])
        # each pair as a complex number, turned by exp(i position f)
        phase = x["positions"].double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
        unit = torch.polar(torch.full_like(phase, factor), phase)
        rd, results = case["rotary_dim"], []
        for t in (x["q"], x["k"]):
            y = t.double().clone()
            lead = y[..., :rd].reshape(*y.shape[:2], rd // 2, 2) if case["interleaved"] else \
                y[..., :rd].reshape(*y.shape[:2], 2, rd // 2).transpose(2, 3)
            z = torch.view_as_real(torch.view_as_complex(lead.contiguous()) * unit)
            y[..., :rd] = (z if case["interleaved"] else z.transpose(2, 3)).reshape(*y.shape[:2], rd)
            results.append(y)
        if case["op"] == "rotary":
            return tuple(results)
        # a token's page is the table entry of its block; walk the tables block by block
        block = case["block_size"]
        total, tables, _ = _tables(x["lengths"], block)
        pools = [torch.zeros(total, case["kv_heads"], block, case["head_dim"], dtype=torch.float64, device="cuda")
                 for _ in range(2)]
        first = 0
        for table, n in zip(tables, x["lengths"]):
            for j, b in enumerate(table):
                m = min(block, n - j * block)
                at = slice(first + j * block, first + j * block + m)
                pools[0][b, :, :m] = results[1][at].transpose(0, 1)
                pools[1][b, :, :m] = x["v"][at].double().transpose(0, 1)
            first += n
        return results[0], results[1], pools[0], pools[1]
    hq, hd = case["q_heads"], case["head_dim"]
    group = hq // case["kv_heads"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    kv0 = q0 = 0
    sizes = [(0, n) for n in x["lengths"]] if case["op"] == "prompt" else list(zip(x["context"], x["nodes"]))
    for c, n in sizes:
        k, v = x["k"][kv0:kv0 + c + n].double(), x["v"][kv0:kv0 + c + n].double()
        hidden = torch.zeros(n, c + n, dtype=torch.bool, device="cuda")
        hidden[:, c:] = ~(torch.arange(n, device="cuda")[:, None] >= torch.arange(n, device="cuda")) \
            if case["op"] == "prompt" else ~x["visible"][q0:q0 + n, :n].cuda()
        for h in range(hq):
            w = x["q"][q0:q0 + n, h].double() @ k[:, h // group].t() / math.sqrt(hd)
            w = torch.exp(w.masked_fill_(hidden, -math.inf) - w.max(-1, keepdim=True).values)
            out[q0:q0 + n, h] = (w @ v[:, h // group]) / w.sum(-1, keepdim=True)
        kv0 += c + n
        q0 += n
    return out
