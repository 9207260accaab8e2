"""pse.rotary / pse.rotary_append against the turn of complex numbers in 64 bits.

Tolerance (fp32): the turn's fraction is rounded to fp32 (2^-26 of a turn, 2 pi
2^-26 in the angle), sincospif is within 2 ulp (2^-23), the factor and the two
products and their sum round once each (4 x 2^-24): below 2^-21 of factor x
(|x1| + |x2|).  A bf16 result has to be the rounding of a value within that
bound.  GPU only."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 8.0},
    "bands": {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 512},
    "yarn": {"type": "yarn", "factor": 16.0, "original": 512},
}


def _plan(*a, **k):
    import pse
    return pse.RotaryPlan(*a, **k)


def reference(x, positions, plan):
    """[T, H, hd] turned in float64, and the bound's |x1| + |x2| (0 where copied)."""
    import pse
    rd, T, H = plan.rotary_dim, x.shape[0], x.shape[1]
    turns = plan.turns.cpu() * 2 * math.pi
    y, size = x.double().cpu().clone(), torch.zeros(x.shape, dtype=torch.float64)
    if rd == 0:
        return y, size
    unit = torch.polar(torch.full((T, 1, rd // 2), plan.factor, dtype=torch.float64),
                       positions.double().cpu()[:, None, None] * turns)
    if plan.interleaved:
        pairs = y[..., :rd].reshape(T, H, rd // 2, 2)
    else:
        pairs = torch.stack((y[..., : rd // 2], y[..., rd // 2: rd]), -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    s = (pairs.abs().sum(-1, keepdim=True) * plan.factor).expand_as(pairs)
    if plan.interleaved:
        y[..., :rd], size[..., :rd] = z.reshape(T, H, rd), s.reshape(T, H, rd)
    else:
        y[..., :rd] = torch.cat((z[..., 0], z[..., 1]), -1)
        size[..., :rd] = torch.cat((s[..., 0], s[..., 1]), -1)
    return y, size


def check(got, x, positions, plan):
    want, size = reference(x, positions, plan)
    bound = size * 2.0 ** -21 + 1e-37 * (size > 0)
    # rounding is monotonic: the result lies between the rounded ends of the bound
    low, high = ((want + s * bound).to(x.dtype) for s in (-1, 1))
    got = got.cpu()
    assert bool(((got >= low) & (got <= high)).all()), float((got.double() - want).abs().max())


def fused(T, hq, hk, hd, dtype, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.randn(T, (hq + 2 * hk) * hd + pad, generator=g, device="cuda").to(dtype)
    h = rows[:, : (hq + 2 * hk) * hd].unflatten(1, (hq + 2 * hk, hd))
    return h[:, :hq], h[:, hq:hq + hk], h[:, hq + hk:]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,hd,rd,interleaved,scaling", [
    (1, 12, 12, 64, 64, False, "none"), (3, 32, 8, 128, 128, False, "bands"), (130, 32, 8, 64, 32, True, "yarn"),
    (257, 5, 1, 80, 32, True, "ntk"), (64, 6, 3, 80, 40, False, "linear"), (33, 3, 3, 96, 48, True, "yarn"),
    (17, 2, 2, 10, 6, False, "none"), (9, 4, 2, 64, 0, False, "none"), (5, 71, 1, 256, 256, True, "none"),
    (4000, 2, 1, 64, 64, False, "ntk"),
])
def test_rotary_matches_complex_turns(dtype, T, hq, hk, hd, rd, interleaved, scaling):
    import pse
    q, k, _ = fused(T, hq, hk, hd, dtype, T + hd)
    plan = _plan(hd, rotary_dim=rd, interleaved=interleaved, scaling=SCALINGS[scaling])
    pos = torch.randint(0, 131072, (T,), device="cuda", dtype=torch.int32)
    qo, ko = pse.rotary(q, k, pos, plan)
    check(qo, q, pos, plan)
    check(ko, k, pos, plan)


def test_extreme_positions_and_no_keys():
    import pse
    q, _, _ = fused(6, 4, 1, 64, torch.float32, 1)
    plan = _plan(64, theta=500000.0)
    pos = torch.tensor([0, -1, -131072, (1 << 31) - 1, -(1 << 31), 1 << 24], dtype=torch.int32, device="cuda")
    qo, none = pse.rotary(q, None, pos, plan)
    assert none is None
    check(qo, q, pos, plan)
    assert torch.equal(qo[0], q[0])  # position 0 turns by nothing


@pytest.mark.parametrize("pad,shift", [(8, 0), (4, 0), (1, 0), (8, 1)])
def test_strides_alignment_and_in_place(pad, shift):
    """Row pitches that are and are not multiples of 16 bytes, a base off
    alignment, heads at a stride of two, and results in place."""
    import pse
    T, hq, hk, hd = 19, 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(pad)
    buf = torch.randn(T, (hq + hk) * hd + pad, generator=g, device="cuda").bfloat16()
    flat = buf[:, shift:shift + (hq + hk) * hd].unflatten(1, (hq + hk, hd))
    q, k = flat[:, :hq:2], flat[:, hq:]
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 977
    plan = _plan(hd, rotary_dim=32)
    q0, k0, all0 = q.clone(), k.clone(), buf.clone()
    qo, ko = pse.rotary(q, k, pos, plan)
    assert torch.equal(buf, all0)
    check(qo, q0, pos, plan)
    q2, k2 = pse.rotary(q, k, pos, plan, q_out=q, k_out=k)
    assert q2 is q and k2 is k
    assert torch.equal(q, qo) and torch.equal(k, ko)
    left = torch.ones_like(buf, dtype=torch.bool)
    lf = left[:, shift:shift + (hq + hk) * hd].unflatten(1, (hq + hk, hd))
    lf[:, :hq:2] = False
    lf[:, hq:] = False
    assert torch.equal(buf[left], all0[left])  # nothing else was written


def test_no_tokens():
    import pse
    plan = _plan(64)
    q = torch.empty(0, 4, 64, device="cuda")
    qo, ko = pse.rotary(q, q[:, :2], torch.empty(0, dtype=torch.int32, device="cuda"), plan)
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,rd,bs,interleaved", [(64, 64, 16, False), (128, 64, 32, True), (80, 40, 4, False)])
def test_append_writes_the_pages_and_nothing_else(dtype, hd, rd, bs, interleaved):
    import pse
    lens, have = [1, 37, 0, 64, 5], [3, 0, 7, 16, 60]
    hq, hk, T = 8, 2, sum(lens)
    cache = pse.PagedKVCache(2, hk, hd, bs, 80, dtype=dtype, max_requests=8)
    ids = [f"r{i}" for i in range(len(lens))]
    g = torch.Generator(device="cuda").manual_seed(hd)
    before = []
    for r, h, n in zip(ids, have, lens):
        cache.create_request(r)
        old = [torch.randn(hk, h + n, hd, generator=g, device="cuda").to(dtype) for _ in range(4)]
        cache.append(r, old[:2], old[2:])
        before.append(old)
    q, k, v = fused(T, hq, hk, hd, dtype, bs, pad=8)
    plan = _plan(hd, rotary_dim=rd, interleaved=interleaved)
    slots = cache.slots_tensor(ids).repeat_interleave(torch.tensor(lens, device="cuda"))
    cpos = torch.cat([torch.arange(h, h + n, device="cuda", dtype=torch.int32) for h, n in zip(have, lens)])
    pos = cpos * 3 + 1  # the rotary position need not be the cache's
    k_out = torch.empty(T, hk, hd, dtype=dtype, device="cuda")
    qo = pse.rotary_append(q, k, v, pos, plan, cache, 1, slots, cpos, k_out=k_out)
    want_q, want_k = pse.rotary(q, k, pos, plan)
    assert torch.equal(qo, want_q) and torch.equal(k_out, want_k)
    kb, vb, _, _ = cache.gather(ids)
    t = 0
    for i, (h, n) in enumerate(zip(have, lens)):
        for layer in (0, 1):
            wk, wv = before[i][layer].clone(), before[i][2 + layer].clone()
            if layer == 1:
                wk[:, h:], wv[:, h:] = want_k[t:t + n].transpose(0, 1), v[t:t + n].transpose(0, 1)
            assert torch.equal(kb[layer][i, :, : h + n], wk) and torch.equal(vb[layer][i, :, : h + n], wv)
        t += n


def test_append_drops_tokens_without_a_block():
    import pse
    cache = pse.PagedKVCache(1, 2, 64, 16, 4, max_requests=2, max_blocks_per_request=4)
    cache.create_request("a")
    cache.append("a", [torch.zeros(2, 20, 64)], [torch.zeros(2, 20, 64)])
    pools = cache.k_pool.clone(), cache.v_pool.clone()
    q, k, v = fused(5, 4, 2, 64, torch.float32, 3)
    s = cache.slot("a")
    slots = torch.tensor([s, s, -1, 99, s], dtype=torch.int32, device="cuda")
    cpos = torch.tensor([32, 1 << 30, 0, 0, -1], dtype=torch.int32, device="cuda")
    plan = _plan(64)
    qo = pse.rotary_append(q, k, v, cpos, plan, cache, 0, slots, cpos)
    check(qo, q, cpos, plan)
    assert torch.equal(cache.k_pool, pools[0]) and torch.equal(cache.v_pool, pools[1])


def test_refusals():
    import pse
    plan = _plan(64)
    q, k, v = fused(4, 4, 2, 64, torch.float32, 0)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q.half()), dict(k=k[:3]), dict(k=k.bfloat16()),
                dict(pos=pos.long()), dict(pos=pos[:3]), dict(pos=pos.cpu()), dict(q=q.transpose(1, 2))):
        a = dict(q=q, k=k, pos=pos)
        a.update(bad)
        with pytest.raises(ValueError):
            pse.rotary(a["q"], a["k"], a["pos"], plan)
    with pytest.raises(ValueError):
        pse.rotary(q, k, pos, plan, q_out=torch.empty(4, 3, 64, device="cuda"))
    for kw in (dict(head_dim=63), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=3),
               dict(head_dim=64, theta=0.0), dict(head_dim=64, scaling={"type": "other"}),
               dict(head_dim=64, scaling={"type": "linear"}), dict(head_dim=64, scaling={"type": "linear", "factor": -1.0})):
        with pytest.raises(ValueError):
            _plan(**kw)
    cache = pse.PagedKVCache(1, 2, 64, 16, 4)
    with pytest.raises(ValueError):
        pse.rotary_append(q, k, v, pos, plan, cache, 1, pos, pos)
    with pytest.raises(ValueError):
        pse.rotary_append(q.bfloat16(), k.bfloat16(), v.bfloat16(), pos, plan, cache, 0, pos, pos)
