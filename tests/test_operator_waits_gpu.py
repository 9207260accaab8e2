"""What follows an expired wait in the tensor-core kernels of packed prompts and
token trees: with no try allowed the consumers give up while the first copies,
which need no wait, are on their way; the kernel lets those end, sets the status
bit and returns, and the next call is right.  Nothing hangs or faults: every
wait is bounded.  GPU only."""
from __future__ import annotations

import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def no_tries():
    from pse import _native as N
    N.call("pse_attention_wait_tries", 0)
    try:
        yield
    finally:
        N.call("pse_attention_wait_tries", -1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[37], [1000, 17, 700], [300] * 60], ids=["one", "three", "many"])
def test_prompts(hd, lens):
    import pse
    g = torch.Generator(device="cuda").manual_seed(hd)
    q, k, v = (torch.randn(sum(lens), h, hd, generator=g, device="cuda").bfloat16() for h in (8, 4, 4))
    p = pse.PackedPrompts(lens, 8, 4)
    want = pse.prompt_attention(q, k, v, p)
    p.check_status()
    for _ in range(3):
        with no_tries():
            pse.prompt_attention(q, k, v, p)
        with pytest.raises(RuntimeError, match=r"status 32\b"):
            p.check_status()
        got = pse.prompt_attention(q, k, v, p)
        p.check_status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [9, 70], ids=["one stream", "two streams"])
@pytest.mark.parametrize("rows", [1, 40])
def test_trees(hd, nodes, rows):
    import pse
    ctx = [17 + 61 * i for i in range(rows)]
    cache = pse.PagedKVCache(1, 2, hd, 16, sum((c + nodes + 15) // 16 for c in ctx), dtype=torch.bfloat16,
                             max_requests=rows, max_blocks_per_request=(max(ctx) + nodes + 15) // 16)
    g = torch.Generator(device="cuda").manual_seed(hd)
    ids = [f"r{i}" for i in range(rows)]
    for r, c in zip(ids, ctx):
        cache.create_request(r)
        cache.append(r, *([torch.randn(2, c + nodes, hd, generator=g, device="cuda")] for _ in range(2)))
    q = torch.randn(rows * nodes, 4, hd, generator=g, device="cuda").bfloat16()
    trees = pse.tree_masks(torch.arange(-1, nodes - 1, dtype=torch.int32, device="cuda").repeat(rows), [nodes] * rows)
    args = (q, cache, 0, cache.slots_tensor(ids), torch.tensor(ctx, dtype=torch.int32, device="cuda"), trees)
    want = pse.token_tree_attention(*args)
    cache.check_status("the first call")
    for _ in range(3):
        with no_tries():
            pse.token_tree_attention(*args)
        with pytest.raises(RuntimeError, match="wait expired"):
            cache.check_status("the call without tries")
        got = pse.token_tree_attention(*args)
        cache.check_status("the call after")
        assert torch.equal(got, want)
