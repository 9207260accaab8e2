"""pse.token_tree_attention and pse.tree_masks against plain evaluations in 64
bits (tolerances as derived in test_prompt_attention_gpu.py: the same
arithmetic, other masks; a request split over thread blocks joins fp32 partial
results, some 2^-24 more).  GPU only."""
from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def random_parents(rng, n, chainy=0.7):
    out = []
    for i in range(n):
        if i == 0 or rng.random() < 0.1:
            out.append(-1)
        else:
            out.append(i - 1 if rng.random() < chainy else rng.randrange(-1, i))
    return out


def ancestor_rows(parents, width):
    m = torch.zeros(len(parents), width, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def words(visible):
    bits = visible.view(visible.shape[0], -1, 64).long()
    return (bits << torch.arange(64)).sum(-1)


class Case:
    def __init__(self, ctx, nodes, hq, hk, hd, bs, dtype, seed, visible=None, stale=None, pad=0):
        import pse
        rng = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.nodes, self.hq, self.hk, self.hd = ctx, nodes, hq, hk, hd
        width = 64 * max(1, (max(nodes, default=0) + 63) // 64)
        if visible is None:
            parts = [ancestor_rows(random_parents(rng, n), width) for n in nodes]
            visible = torch.cat(parts) if parts else torch.zeros(0, width, dtype=torch.bool)
        self.visible = visible
        every = [c + n for c, n in zip(ctx, nodes)]
        blocks = sum((n + bs - 1) // bs for n in every) + 3
        self.cache = pse.PagedKVCache(2, hk, hd, bs, blocks, dtype=dtype, max_requests=max(1, len(ctx)),
                                      max_blocks_per_request=max([1] + [(n + bs - 1) // bs for n in every]))
        if stale is not None:
            self.cache.k_pool.fill_(stale)
            self.cache.v_pool.fill_(stale)
        self.k = [torch.randn(hk, n, hd, generator=g, device="cuda").to(dtype) for n in every]
        self.v = [torch.randn(hk, n, hd, generator=g, device="cuda").to(dtype) for n in every]
        self.ids = [f"r{i}" for i in range(len(ctx))]
        for r in self.ids:
            self.cache.create_request(r)
        self.fill()
        N = sum(nodes)
        self.q = torch.randn(N, hq * hd + pad, generator=g, device="cuda").to(dtype)[:, : hq * hd].unflatten(1, (hq, hd))
        self.trees = pse.TokenTrees(words(visible).cuda(), nodes)
        self.context = torch.tensor(ctx, dtype=torch.int32, device="cuda")

    def fill(self):
        for r, k, v in zip(self.ids, self.k, self.v):
            if k.shape[1]:
                self.cache.append(r, [torch.zeros_like(k), k], [torch.zeros_like(v), v])

    def run(self, **kw):
        import pse
        slots = self.cache.slots_tensor(self.ids)
        out = pse.token_tree_attention(self.q, self.cache, 1, slots, self.context, self.trees, **kw)
        self.cache.check_status("test")
        return out

    def reference(self, scale):
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        g, t = self.hq // self.hk, 0
        for c, n, k, v in zip(self.ctx, self.nodes, self.k, self.v):
            if n == 0:
                continue
            see = torch.cat((torch.ones(n, c, dtype=torch.bool), self.visible[t:t + n, :n]), 1).cuda()
            qq = self.q[t:t + n].double().transpose(0, 1)
            kk, vv = k.double().repeat_interleave(g, 0), v.double().repeat_interleave(g, 0)
            s = (qq @ kk.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)  # a row that sees nothing: zeros
            A = p @ vv.abs()
            if self.q.dtype == torch.float32:
                dot = (qq.abs() @ kk.abs().transpose(1, 2) * scale).amax(-1, keepdim=True)
                A = A * (2 * (self.hd + 4) * 2.0 ** -24 * dot + (c + n + 32) * 2.0 ** -24)
            else:
                A = A * (2.0 ** -7 + 2.0 ** -10)
            out[t:t + n], bound[t:t + n] = (p @ vv).transpose(0, 1), A.transpose(0, 1)
            t += n
        return out, bound

    def check(self, scale=None, **kw):
        got = self.run(scale=scale, **kw)
        want, bound = self.reference(1 / math.sqrt(self.hd) if scale is None else scale)
        err = (got.double() - want).abs()
        assert bool((err <= bound + 1e-37).all()), float((err - bound).max())
        return got


SHAPES = [
    ([0], [1]), ([1], [1]), ([5, 0, 130], [3, 7, 0]), ([127, 128, 129, 255], [1, 64, 2, 33]),
    ([300, 17, 1000, 64], [8, 64, 1, 20]), ([4000], [60]), ([0, 0], [64, 1]), ([63, 62, 61], [1, 2, 3]),
    ([40] * 30, [5] * 30), ([2000, 3, 700], [130, 200, 1]),
]


@pytest.mark.parametrize("hq,hk,hd,bs", [(12, 12, 64, 16), (32, 8, 64, 32), (32, 8, 128, 64), (4, 1, 128, 16)])
@pytest.mark.parametrize("ctx,nodes", SHAPES, ids=lambda x: "-".join(map(str, x[:4])))
def test_bf16_matches_reference(ctx, nodes, hq, hk, hd, bs):
    Case(ctx, nodes, hq, hk, hd, bs, torch.bfloat16, sum(ctx) + bs).check()


@pytest.mark.parametrize("hq,hk,hd,bs", [(12, 12, 64, 16), (8, 2, 33, 5), (2, 1, 256, 8)])
@pytest.mark.parametrize("ctx,nodes", SHAPES[:8], ids=lambda x: "-".join(map(str, x[:4])))
def test_fp32_matches_reference(ctx, nodes, hq, hk, hd, bs):
    Case(ctx, nodes, hq, hk, hd, bs, torch.float32, sum(ctx) + bs).check()


@pytest.mark.parametrize("hq,hk,hd,bs", [(6, 2, 96, 16), (5, 1, 64, 4), (7, 7, 128, 8), (64, 1, 64, 16), (40, 1, 128, 32),
                                         (3, 3, 64, 128), (8, 8, 128, 128), (2, 2, 64, 48)])
def test_other_heads_and_pages(hq, hk, hd, bs):
    Case([200, 0, 31], [9, 4, 17], hq, hk, hd, bs, torch.bfloat16, hq).check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 200, 700])
def test_many_and_few_requests(hd, rows):
    """Cuts of the work line inside items, whole items per block, more rows than threads."""
    rng = random.Random(rows)
    top = 6000 if rows <= 3 else 400
    ctx = [rng.randrange(0, top) for _ in range(rows)]
    nodes = [rng.randrange(0, 10) for _ in range(rows)]
    nodes[0] = 10
    Case(ctx, nodes, 8, 2, hd, 16, torch.bfloat16, rows).check()


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_masks_that_hide_everything(hd, dtype):
    """No context and an empty mask: zeros; bits past the tree: no keys; masks
    that are no tree at all."""
    nodes = [3, 5, 70]
    vis = torch.rand(78, 128, generator=torch.Generator().manual_seed(1)) < 0.3
    vis[0], vis[4], vis[40] = False, False, False
    c = Case([0, 0, 9], nodes, 4, 2, hd, 16, dtype, 3, visible=vis)
    got = c.check()
    assert bool((got[0] == 0).all()) and bool((got[4] == 0).all()) and bool((got[40] != 0).any())


@pytest.mark.parametrize("stale", [math.nan, math.inf])
@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_stale_pages_and_poisoned_siblings(stale, hd, dtype):
    """What stands in the pool past a row's nodes, or in nodes that a node does
    not see, does not reach it; what it sees does."""
    c = Case([20, 0, 130], [6, 3, 40], 8, 2, hd, 16, dtype, 5, stale=stale)
    clean = c.check()
    c2 = Case([20, 0, 130], [6, 3, 40], 8, 2, hd, 16, dtype, 5, stale=stale)
    for r in c2.ids:
        c2.cache.truncate(r, 0)
    c2.v[2][0, 130 + 4, 1] = math.inf
    c2.v[2][0, 130 + 9, 2] = math.nan
    c2.k[2][0, 130 + 20] = math.nan
    c2.fill()
    got = c2.run()
    first = 9
    sees = c2.visible[first:]
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[first:, :4, 1] |= sees[:, 4].cuda()[:, None]
    hit[first:, :4, 2] |= sees[:, 9].cuda()[:, None]
    hit[first:, :4] |= sees[:, 20].cuda()[:, None, None]
    assert bool((~torch.isfinite(got[hit])).all()) and hit.any()
    # the rest of the poisoned K/V head may round otherwise where a tile is taken apart
    assert torch.equal(got[~hit], clean[~hit])


def test_invalid_rows_give_zeros():
    import pse
    c = Case([10, 20, 30], [2, 3, 4], 4, 2, 64, 16, torch.bfloat16, 6)
    want = c.run()
    slots = c.cache.slots_tensor(c.ids)
    slots[1] = 99
    got = pse.token_tree_attention(c.q, c.cache, 1, slots, c.context, c.trees)
    assert bool((got[2:5] == 0).all()) and torch.equal(got[:2], want[:2]) and torch.equal(got[5:], want[5:])
    ctx = c.context.clone()
    ctx[0], ctx[2] = -5, 1 << 30
    got = pse.token_tree_attention(c.q, c.cache, 1, c.cache.slots_tensor(c.ids), ctx, c.trees)
    assert bool((got[:2] == 0).all()) and bool((got[5:] == 0).all()) and torch.equal(got[2:5], want[2:5])


@pytest.mark.parametrize("hd", [64, 128])
def test_strides_and_output(hd):
    c = Case([100, 7], [12, 5], 8, 4, hd, 16, torch.bfloat16, 7, pad=8)
    first = c.check()
    buf = torch.full((17, 8 * hd + 4), 3.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, : 8 * hd].unflatten(1, (8, hd))
    assert torch.equal(c.check(out=out), first) and bool((buf[:, 8 * hd:] == 3.0).all())
    c.q = torch.randn(17, 8 * hd + 1, device="cuda").bfloat16()[:, 1:].unflatten(1, (8, hd))
    c.check()


def test_one_chain_is_causal_attention():
    """A tree that is one chain: the paged attention of consecutive tokens."""
    from pse import _native as N
    nodes = [5, 5, 5]
    vis = torch.cat([ancestor_rows([-1, 0, 1, 2, 3], 64)] * 3)
    c = Case([50, 3, 200], nodes, 8, 2, 64, 16, torch.bfloat16, 8, visible=vis)
    got = c.check()
    out = torch.empty(15, 8 * 64, dtype=torch.bfloat16, device="cuda")
    slots = c.cache.slots_tensor(c.ids)
    ws = torch.zeros(N.size_call("pse_paged_attention_workspace", 3, 5, 8, 2, 64, 256), dtype=torch.uint8, device="cuda")
    qc = c.q.reshape(15, -1).contiguous()
    N.call("pse_paged_attention", c.cache.state, c.cache.layer(1), qc.data_ptr(), 512, out.data_ptr(), 512,
           slots.data_ptr(), c.context.data_ptr(), 3, 5, 8, 0.125, 256, None, ws.data_ptr(), ws.numel(), N.stream_ptr())
    want, bound = c.reference(0.125)
    assert bool(((out.view(15, 8, 64).double() - want).abs() <= bound).all())
    assert bool(((out.view(15, 8, 64).double() - got.double()).abs() <= 2 * bound).all())


def test_repeats_streams_and_graph_replay():
    """The same bits on every call, on another stream, and from a graph whose
    lengths change between replays."""
    import pse
    import pse._native as N
    c = Case([900, 40, 2500], [30, 2, 11], 16, 4, 128, 32, torch.bfloat16, 9)
    first = c.check()
    for _ in range(3):
        assert torch.equal(c.run(), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = c.run()
    torch.cuda.synchronize()
    assert torch.equal(other, first)
    slots = c.cache.slots_tensor(c.ids)
    ctx, out = c.context.clone(), torch.empty_like(first)
    g = torch.cuda.CUDAGraph()
    with N.graph_capture(g):
        pse.token_tree_attention(c.q, c.cache, 1, slots, ctx, c.trees, out=out)
    g.replay()
    assert torch.equal(out, first)
    ctx.copy_(torch.tensor([100, 40, 1], dtype=torch.int32))
    want = pse.token_tree_attention(c.q, c.cache, 1, slots, ctx, c.trees)
    for _ in range(2):
        g.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("counts", [[1], [0, 5, 0], [64, 65, 1], [200, 3, 130]])
def test_tree_masks(counts):
    import pse
    rng = random.Random(len(counts))
    parents = [random_parents(rng, n) for n in counts]
    width = 64 * max(1, (max(counts) + 63) // 64)
    flat = torch.tensor([p for t in parents for p in t], dtype=torch.int32, device="cuda")
    trees = pse.tree_masks(flat, counts)
    want = torch.cat([ancestor_rows(t, width) for t in parents if t])
    assert torch.equal(trees.masks.cpu(), words(want))
    assert torch.equal(trees.depths.cpu().long(), want.sum(-1) - 1)
    # a parent that does not precede its child ends the walk
    bad = flat.clone()
    bad[0] = 7
    assert pse.tree_masks(bad, counts).depths[0] == 0


def test_refusals():
    import pse
    c = Case([10], [4], 4, 2, 64, 16, torch.bfloat16, 1)
    slots = c.cache.slots_tensor(c.ids)
    ok = dict(q=c.q, layer=0, slots=slots, context=c.context, trees=c.trees)
    for bad in (dict(q=c.q[:3]), dict(q=c.q.float()), dict(q=c.q[:, :3]), dict(layer=2), dict(slots=slots.long()),
                dict(context=c.context[:0]), dict(q=c.q[..., :32]), dict(q=c.q.cpu())):
        a = {**ok, **bad}
        with pytest.raises(ValueError):
            pse.token_tree_attention(a["q"], c.cache, a["layer"], a["slots"], a["context"], a["trees"])
    m = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    for a in ((m, [3]), (m, [5, -1]), (m.int(), [4]), (m.cpu(), [4]), (torch.zeros(65, 1, dtype=torch.int64, device="cuda"), [65])):
        with pytest.raises(ValueError):
            pse.TokenTrees(*a)
    with pytest.raises(ValueError):
        pse.tree_masks(torch.zeros(3, dtype=torch.int32), [3])
    with pytest.raises(RuntimeError):
        pse.token_tree_attention(c.q, c.cache, 0, slots, c.context, c.trees,
                                 workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))


def test_refusals_of_kept_buffers():
    """A workspace or offsets that the kernel cannot use are refused before the launch."""
    import pse
    c = Case([5, 9], [3, 2], 4, 2, 64, 16, torch.bfloat16, 1)
    size = pse.token_tree.token_tree_workspace(64, "cuda").numel()
    for bad in (torch.zeros(size, dtype=torch.uint8), torch.zeros(size, dtype=torch.int32, device="cuda"),
                torch.zeros(2 * size, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError):
            c.run(workspace=bad)
    for bad in (torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32),
                torch.zeros(3, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError):
            pse.TokenTrees(c.trees.masks, c.nodes, offsets=bad)


@pytest.mark.parametrize("group,nodes", [(17, [1]), (32, [1, 1]), (64, [2, 0, 1]), (2, [16, 3]), (2, [17, 16])])
def test_few_rows_of_large_groups(group, nodes):
    """The CUDA-core kernel's blocks hold whole groups, and any number of rows around its two sizes."""
    Case([70] * len(nodes), nodes, 2 * group, 2, 40, 8, torch.float32, group).check()


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32), (80, torch.bfloat16)])
def test_a_visible_infinity_of_no_weight_reaches_the_row(hd, dtype):
    """A key that a row sees counts, however far its score lies below the
    largest: 0 x inf is NaN, wherever the work is cut."""
    ctx = 3000
    c = Case([ctx], [3], 2, 2, hd, 16, dtype, 2)
    c.cache.truncate("r0", 0)
    c.q.fill_(1.0)
    c.k[0].zero_()
    c.k[0][:, ctx] = 400.0 / math.sqrt(hd)  # the first node, an ancestor of all: scores of 400
    c.visible[:, 0] = True
    c.trees = __import__("pse").TokenTrees(words(c.visible).cuda(), [3])
    c.v[0][0, 5, 1], c.v[0][1, 7, 2] = math.nan, math.inf
    c.fill()
    got = c.run()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, 0, 1] = bad[:, 1, 2] = True
    assert not torch.isfinite(got[bad]).any() and torch.isfinite(got[~bad]).all()


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32), (80, torch.bfloat16)])
@pytest.mark.parametrize("at", [5, 41])
def test_an_infinity_of_no_weight_in_a_tile_with_a_mask(at, hd, dtype):
    """The same beside hidden keys: in the context, and in a node that the next ones see and the one before does not."""
    c = Case([40], [4], 2, 2, hd, 16, dtype, 2, visible=ancestor_rows([-1, -1, 1, 2], 64))
    c.cache.truncate("r0", 0)
    c.q.fill_(1.0)
    c.k[0].zero_()
    c.k[0][:, 7] = 400.0 / math.sqrt(hd)  # a key of the context, which all see
    c.v[0][0, at, 1], c.v[0][1, at, 2] = math.nan, math.inf
    c.fill()
    got = c.run()
    bad = torch.zeros_like(got, dtype=torch.bool)
    first = 0 if at < 40 else 1
    bad[first:, 0, 1] = bad[first:, 1, 2] = True
    assert not torch.isfinite(got[bad]).any() and torch.isfinite(got[~bad]).all()
