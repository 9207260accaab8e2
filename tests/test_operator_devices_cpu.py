"""Which device the packed operators launch on.  CPU only: tensors that say they
are on a GPU, a stand-in for the current device, and library functions that
are recorded, not called."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


class OnGpu(torch.Tensor):
    """A CPU tensor that gives GPU 1 as its device."""
    is_cuda = True

    def get_device(self):
        return 1


def gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


class Calls:
    """The five launches, over tensors of GPU 1, with `current` the current device."""

    def __init__(self, monkeypatch, current):
        from pse import _native
        self.made = []
        monkeypatch.setattr(_native, "_current_device", lambda: current)
        monkeypatch.setattr(_native, "_raw_stream", lambda device: 1000 + device)
        monkeypatch.setattr(_native, "call", lambda name, *a: self.made.append((name, a[-1])))
        monkeypatch.setattr(_native, "load", lambda: None)
        monkeypatch.setattr(_native, "fn", lambda name: self.record(name))
        index = torch.device("cuda", 1)
        self.q, self.kv, self.i = gpu(3, 4, 8), gpu(3, 2, 8), gpu(3, dtype=torch.int32)
        self.plan = SimpleNamespace(head_dim=8, index=1, spec=None, fn=self.record("rotary"),
                                    append_fn=self.record("append"))
        self.cache = SimpleNamespace(head_dim=8, n_heads=2, n_layers=1, dtype=torch.float32, device=index, state=None,
                                     layer=lambda i: None)
        self.prompts = SimpleNamespace(index=1, tokens=3, q_heads=4, kv_heads=2, fn=self.record("prompts"),
                                       _plan_ptr=0, n_cta=1, n_items=1, _status_ptr=0)
        self.trees = SimpleNamespace(index=1, nodes=3, counts=[3], max_nodes=3, words=1, _offsets_ptr=0, _masks_ptr=0,
                                     fn=self.record("trees"))

    def record(self, name):
        def fn(*a):
            self.made.append((name, a[-1]))
            return 0
        return fn

    def make(self, what):
        import pse
        from pse import token_tree
        if what == "rotary":
            pse.rotary(self.q, self.kv, self.i, self.plan)
        elif what == "append":
            pse.rotary_append(self.q, self.kv, self.kv, self.i, self.plan, self.cache, 0, self.i, self.i)
        elif what == "prompts":
            pse.prompt_attention(self.q, self.kv, self.kv, self.prompts)
        elif what == "trees":
            pse.token_tree_attention(self.q, self.cache, 0, self.i[:1], self.i[:1], self.trees,
                                     workspace=gpu(16, dtype=torch.uint8))
        else:
            token_tree.TokenTrees = lambda *a: None
            pse.tree_masks(self.i, [3])


@pytest.mark.parametrize("what", ["rotary", "append", "prompts", "trees", "masks"])
def test_launches_only_on_the_tensors_device(monkeypatch, what):
    """With another device current the kernel would run over addresses of a GPU
    that it is not on: refused before anything is launched."""
    from pse import token_tree
    monkeypatch.setattr(token_tree, "TokenTrees", token_tree.TokenTrees)
    calls = Calls(monkeypatch, current=0)
    with pytest.raises(ValueError, match="GPU 0 is current"):
        calls.make(what)
    assert calls.made == []
    calls = Calls(monkeypatch, current=1)
    calls.make(what)
    assert [stream for _, stream in calls.made] == [1001]
