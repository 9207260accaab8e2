"""Outputs given by the caller of the packed operators: each element needs a
place of its own, whatever the order of the axes.  CPU only (the checks run
before a launch)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

T, H, D = 6, 4, 8
GOOD = {
    "contiguous": lambda: torch.zeros(T, H, D),
    "padded": lambda: torch.zeros(T, H * D + 3)[:, : H * D].unflatten(1, (H, D)),
    "heads first": lambda: torch.zeros(H, T, D).transpose(0, 1),
    "every second head": lambda: torch.zeros(T, 2 * H, D)[:, ::2],
    "every second token": lambda: torch.zeros(2 * T, H, D)[::2],
    "half heads": lambda: torch.zeros(T, H, 2 * D)[..., :D],
    "heads first, padded": lambda: torch.zeros(H, T + 2, D + 1)[:, :T, :D].transpose(0, 1),
}
BAD = {
    "one token for all": lambda: torch.zeros(1, H, D).expand(T, H, D),
    "one head for all": lambda: torch.zeros(T, 1, D).expand(T, H, D),
    "sliding tokens": lambda: torch.zeros(T * H * D).as_strided((T, H, D), (D, D, 1)),
    "sliding heads": lambda: torch.zeros(T * H * D).as_strided((T, H, D), (H * D, D - 1, 1)),
    "heads first, sliding": lambda: torch.zeros(T * H * D).as_strided((T, H, D), (D, T * D - 1, 1)),
}


def _given(monkeypatch, what, out):
    """`out` given to the operator as its output; the launches made."""
    import pse
    from pse import _native
    made = []
    launch = lambda *a: made.append(a) or 0  # noqa: E731
    monkeypatch.setattr(_native, "_current_device", lambda: -1)  # what a CPU tensor gives as its device
    monkeypatch.setattr(_native, "_raw_stream", lambda device: 0)
    q, kv, i = torch.zeros(T, H, D), torch.zeros(T, H, D), torch.zeros(T, dtype=torch.int32)
    plan = SimpleNamespace(head_dim=D, index=-1, spec=None, fn=launch, append_fn=launch)
    cache = SimpleNamespace(head_dim=D, n_heads=H, n_layers=1, dtype=torch.float32, device=SimpleNamespace(index=-1),
                            state=None, layer=lambda j: None)
    if what in ("q_out", "k_out"):
        pse.rotary(q, kv, i, plan, **{what: out})
    elif what == "append":
        pse.rotary_append(q, kv, kv, i, plan, cache, 0, i, i, k_out=out)
    elif what == "prompts":
        pse.prompt_attention(q, kv, kv, SimpleNamespace(index=-1, tokens=T, q_heads=H, kv_heads=H, fn=launch, _plan_ptr=0,
                                                        n_cta=1, n_items=1, _status_ptr=0), out=out)
    else:
        trees = SimpleNamespace(index=-1, nodes=T, counts=[T], max_nodes=T, words=1, _offsets_ptr=0, _masks_ptr=0, fn=launch)
        pse.token_tree_attention(q, cache, 0, i[:1], i[:1], trees, out=out, workspace=torch.zeros(16, dtype=torch.uint8))
    return len(made)


@pytest.mark.parametrize("what", ["q_out", "k_out", "append", "prompts", "trees"])
def test_outputs_that_overlap_themselves_are_refused(monkeypatch, what):
    for name, out in BAD.items():
        with pytest.raises(ValueError, match="overlaps itself"):
            _given(monkeypatch, what, out())
            pytest.fail(name)
    for name, out in GOOD.items():
        assert _given(monkeypatch, what, out()) == 1, name


@pytest.mark.parametrize("shape,strides,fine", [
    ((1, 4, 8), (0, 8, 1), True), ((6, 1, 8), (8, 0, 1), True), ((1, 1, 8), (0, 0, 1), True), ((0, 4, 8), (0, 0, 1), True),
    ((6, 0, 8), (0, 0, 1), True), ((1, 4, 8), (32, 0, 1), False), ((6, 1, 8), (0, 8, 1), False),
    ((6, 1, 8), (7, 8, 1), False)])
def test_strides_of_axes_of_one_do_not_matter(shape, strides, fine):
    from pse.rotary import written_view
    args = ("out", torch.zeros(400).as_strided(shape, strides), shape[0], shape[1], 8, torch.float32, -1)
    if fine:
        written_view(*args)
    else:
        with pytest.raises(ValueError, match="overlaps itself"):
            written_view(*args)
