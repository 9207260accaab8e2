"""The packed operators on a cache whose device was given without an index.  GPU only."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("device", [None, "cuda", torch.device("cuda"), "cuda:0", 0])
def test_a_cache_of_the_current_device_is_taken(device):
    import pse
    cache = pse.PagedKVCache(1, 2, 64, 16, 4, device=device)
    assert cache.device == torch.device("cuda", 0) == cache.k_pool.device
    plan = pse.RotaryPlan(64, device="cuda")
    cache.create_request("a")
    cache.append("a", [torch.zeros(2, 3, 64)], [torch.zeros(2, 3, 64)])
    q, k, v = torch.randn(3, 4, 64, device="cuda"), torch.randn(3, 2, 64, device="cuda"), torch.randn(3, 2, 64, device="cuda")
    at = torch.arange(3, dtype=torch.int32, device="cuda")
    turned = pse.rotary_append(q, k, v, at, plan, cache, 0, cache.slots_tensor(["a"]).expand(3).contiguous(), at)
    assert torch.equal(turned, pse.rotary(q, None, at, plan)[0])
    trees = pse.tree_masks(torch.tensor([-1, 0, 1], dtype=torch.int32, device="cuda"), [3])
    context = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = pse.token_tree_attention(turned, cache, 0, cache.slots_tensor(["a"]), context, trees)
    # the first node sees itself alone
    assert torch.allclose(out[0], v[0].repeat_interleave(2, 0))
