"""pse.prompt_attention against the masked softmax in 64 bits.

Tolerances, per element against A = sum_j p_j |v_j|.  bf16 (unit roundoff 2^-8):
weights rounded to bf16 move the result by 2^-8 A at most and the result rounds
once (2^-8 |o| <= 2^-8 A); the fp32 scores, exponentials and sums add well under
2^-10 A: (2^-7 + 2^-10) A.
fp32: a score of hd products is off by (hd + 4) 2^-24 sum |q||k| scale, which
moves the normalised weights by twice that, and n terms are summed: (2 max_j
(hd + 4) 2^-24 sum |q||k| scale + (n + 16) 2^-24) A.  GPU only."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(lens, hq, hk, hd, dtype, seed, pad=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens)
    rows = (torch.randn(T, (hq + 2 * hk) * hd + pad, generator=g, device="cuda") * size).to(dtype)
    h = rows[:, : (hq + 2 * hk) * hd].unflatten(1, (hq + 2 * hk, hd))
    return h[:, :hq], h[:, hq:hq + hk], h[:, hq + hk:]


def reference(q, k, v, lens, scale):
    """(out, bound of an fp32 / bf16 evaluation) in float64."""
    T, hq, hd = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(T, hq, hd, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    t = 0
    for n in lens:
        qq, kk, vv = (x[t:t + n].double().transpose(0, 1) for x in (q, k, v))
        kk, vv = kk.repeat_interleave(g, 0), vv.repeat_interleave(g, 0)
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        s = (qq @ kk.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1)
        # 0 x inf is no part of a hidden key
        o = p @ torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0)
        A = p @ torch.nan_to_num(vv, nan=0.0, posinf=0.0, neginf=0.0).abs()
        if q.dtype == torch.float32:
            dot = (qq.abs() @ kk.abs().transpose(1, 2) * abs(scale)).masked_fill(hidden, 0).amax(-1, keepdim=True)
            A = A * (2 * (hd + 4) * 2.0 ** -24 * dot + (n + 16) * 2.0 ** -24)
        else:
            A = A * (2.0 ** -7 + 2.0 ** -10)
        out[t:t + n], bound[t:t + n] = o.transpose(0, 1), A.transpose(0, 1)
        t += n
    return out, bound


def run(q, k, v, lens, **kw):
    import pse
    p = pse.PackedPrompts(lens, q.shape[1], k.shape[1])
    out = pse.prompt_attention(q, k, v, p, **kw)
    p.check_status()
    return out


def check(q, k, v, lens, scale=None, **kw):
    got = run(q, k, v, lens, scale=scale, **kw)
    want, bound = reference(q, k, v, lens, 1 / math.sqrt(q.shape[2]) if scale is None else scale)
    err = (got.double() - want).abs()
    assert bool((err <= bound + 1e-37).all()), float((err - bound).max())
    return got


LENS = [[1], [2, 1, 3], [37], [127, 128, 129], [64, 0, 65, 0], [255, 256, 257, 1], [511, 33], [1000, 17, 700],
        [5] * 40]


@pytest.mark.parametrize("hq,hk,hd", [(12, 12, 64), (32, 8, 64), (8, 1, 128), (6, 2, 128)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:4])))
def test_bf16_matches_reference(lens, hq, hk, hd):
    check(*inputs(lens, hq, hk, hd, torch.bfloat16, sum(lens) + hq), lens)


@pytest.mark.parametrize("hq,hk,hd", [(12, 12, 64), (4, 2, 128), (7, 7, 33), (2, 1, 256)])
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [63, 0, 64, 65], [300, 17]], ids=lambda x: "-".join(map(str, x)))
def test_fp32_matches_reference(lens, hq, hk, hd):
    check(*inputs(lens, hq, hk, hd, torch.float32, sum(lens) + hq), lens)


@pytest.mark.parametrize("hq,hk,hd", [(3, 3, 96), (5, 1, 80), (4, 4, 16), (130, 1, 64), (20, 4, 64), (24, 8, 128),
                                      (128, 1, 128), (129, 3, 64)])
def test_other_heads_and_groups(hq, hk, hd):
    lens = [70, 1, 140]
    check(*inputs(lens, hq, hk, hd, torch.bfloat16, hd), lens)


@pytest.mark.parametrize("hd", [64, 128])
def test_long_prompts_and_large_scores(hd):
    """Many key tiles; scores that spread the weights over hundreds of octaves."""
    lens = [3001, 2048]
    check(*inputs(lens, 4, 1, hd, torch.bfloat16, 5, size=3.0), lens)
    check(*inputs(lens, 4, 1, hd, torch.bfloat16, 6), lens, scale=0.01)


@pytest.mark.parametrize("hd", [64, 128])
def test_rising_scores(hd):
    """Keys that grow along the prompt move the running maximum in every tile."""
    lens = [1200]
    q, k, v = (x.clone() for x in inputs(lens, 4, 2, hd, torch.bfloat16, 9))
    q.copy_(q.abs())
    k.copy_(k.abs() * (torch.arange(1200, device="cuda")[:, None, None] / 200).to(k.dtype))
    check(q, k, v, lens)
    check(q, -k, v, lens)


@pytest.mark.parametrize("pad", [8, 1])
@pytest.mark.parametrize("hd", [64, 128])
def test_strides(pad, hd):
    """Row pitches on and off 16 bytes, heads at a stride, an output of its own pitch."""
    lens = [150, 40]
    q, k, v = inputs(lens, 8, 4, hd, torch.bfloat16, 3, pad=pad)
    buf = torch.full((190, 8 * hd + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, : 8 * hd].unflatten(1, (8, hd))
    check(q, k, v, lens, out=out)
    assert bool((buf[:, 8 * hd:] == 7.0).all())
    check(q[:, ::2], k[:, ::2], v[:, ::2], lens)
    wide = torch.randn(190, 4, 2 * hd, device="cuda").bfloat16()
    check(q, wide[..., :hd], wide[..., hd:], lens)


@pytest.mark.parametrize("hq,hk,hd,dtype", [(8, 2, 64, torch.bfloat16), (4, 4, 128, torch.bfloat16),
                                            (4, 2, 64, torch.float32)])
def test_poison_behind_the_mask_stays_there(hq, hk, hd, dtype):
    """Infinities and NaN in later tokens and in other prompts change nothing;
    those that a token sees reach it."""
    lens = [100, 200, 31]
    q, k, v = (x.clone() for x in inputs(lens, hq, hk, hd, dtype, 17))
    clean = run(q, k, v, lens)
    bad = math.nan if dtype == torch.float32 else math.inf
    v[230, 0, 3], v[231, 0, 5], v[232, 0, 7] = bad, -math.inf, math.nan
    k[240, 0], k[250, 0, 0] = math.nan, math.inf
    got = run(q, k, v, lens)
    g = hq // hk
    seen = torch.zeros_like(clean, dtype=torch.bool)
    for t, d in ((230, 3), (231, 5), (232, 7)):
        seen[t:300, :g, d] = True
    assert not torch.isfinite(got[seen]).any()
    assert torch.isnan(got[240:300, :g]).all()
    seen[240:300, :g] = True
    assert torch.equal(got[~seen], clean[~seen])
    if dtype == torch.bfloat16:
        assert bool((got[230:240, :g, 3] == math.inf).all()) and bool((got[231:240, :g, 5] == -math.inf).all())


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32)])
def test_a_row_of_minus_infinity_gives_zero(hd, dtype):
    lens = [70]
    q, k, v = (x.clone() for x in inputs(lens, 2, 2, hd, dtype, 4))
    q[3, 0] = 0
    q[3, 0, 0] = 1
    k[:4, 0, 0] = -math.inf
    got = run(q, k, v, lens)
    assert bool((got[3, 0] == 0).all())


def test_order_of_calls_streams_and_plans():
    """The same call gives the same bits, also on another stream and beside
    another packing."""
    lens = [400, 1, 90]
    q, k, v = inputs(lens, 8, 2, 64, torch.bfloat16, 8)
    first = run(q, k, v, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run(q, k, v, lens)
    run(q, k, v, [491])
    torch.cuda.synchronize()
    assert torch.equal(first, other) and torch.equal(first, run(q, k, v, lens))


def test_captured_in_a_graph():
    import pse
    import pse._native as N
    lens = [77, 300]
    q, k, v = (x.clone() for x in inputs(lens, 8, 2, 64, torch.bfloat16, 12))
    p = pse.PackedPrompts(lens, 8, 2)
    out = pse.prompt_attention(q, k, v, p)
    g = torch.cuda.CUDAGraph()
    with N.graph_capture(g):
        pse.prompt_attention(q, k, v, p, out=out)
    q.copy_(inputs(lens, 8, 2, 64, torch.bfloat16, 13)[0])
    g.replay()
    assert torch.equal(out, pse.prompt_attention(q, k, v, p))


def test_empty():
    import pse
    for lens in ([], [0], [0, 0, 0]):
        q = torch.empty(0, 4, 64, device="cuda")
        assert pse.prompt_attention(q, q[:, :2], q[:, :2], pse.PackedPrompts(lens, 4, 2)).shape == (0, 4, 64)


def test_refusals():
    import pse
    q, k, v = inputs([10], 4, 2, 64, torch.bfloat16, 0)
    p = pse.PackedPrompts([10], 4, 2)
    for a in ((q[:9], k, v), (q, k[:9], v), (q, k, v.float()), (q.half(), k.half(), v.half()), (q[:, :2], k, v),
              (q, k[:, :1], v), (q.cpu(), k.cpu(), v.cpu()), (q, k, v[..., :32]), (q[..., ::2], k[..., ::2], v[..., ::2])):
        with pytest.raises(ValueError):
            pse.prompt_attention(*a, p)
    with pytest.raises(ValueError):
        pse.prompt_attention(q, k, v, p, out=torch.empty(10, 4, 64, device="cuda"))
    for a in (([-1], 4, 2), ([3], 4, 3), ([3], 0, 1), ([1 << 30, 1 << 30], 4, 2)):
        with pytest.raises(ValueError):
            pse.PackedPrompts(*a)


@pytest.mark.parametrize("hd", [64, 128])
def test_many_short_items_behind_a_long_one(hd):
    """Every multiprocessor takes items of two query tiles and then many of one,
    whose second stream has no part in them; the marks of value tiles with
    infinities stay with their own item."""
    lens = [200] * 20 + [100] * 260 + [1] * 40
    hq = hk = 8
    q, k, v = (x.clone() for x in inputs(lens, hq, hk, hd, torch.bfloat16, 21))
    clean = run(q, k, v, lens)
    check(q, k, v, lens)
    seen, t = torch.zeros_like(clean, dtype=torch.bool), 0
    for i, n in enumerate(lens):
        at = t + n * 3 // 4  # in the second tile of a long prompt
        if i % 3 == 0:
            v[at, i % hk, i % hd] = math.inf
            seen[at:t + n, i % hk, i % hd] = True
        t += n
    got = run(q, k, v, lens)
    assert bool((got[seen] == math.inf).all()) and torch.equal(got[~seen], clean[~seen])


@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float32), (80, torch.bfloat16)])
def test_a_visible_infinity_of_no_weight_reaches_the_row(hd, dtype):
    """A key that a token sees counts, however far its score lies below the largest: 0 x inf is NaN."""
    lens = [200, 30]
    q, k, v = (x.clone() for x in inputs(lens, 2, 2, hd, dtype, 2))
    q.fill_(1.0)
    k.zero_()
    k[0] = k[200] = 400.0 / math.sqrt(hd)  # scores of 400 beside zeros
    seen = torch.zeros_like(q, dtype=torch.bool)
    for t, h, d in ((5, 0, 1), (150, 1, 2), (210, 0, 3)):
        v[t, h, d] = math.inf if t == 150 else math.nan
        seen[t:200 if t < 200 else 230, h, d] = True
    got = run(q, k, v, lens)
    assert not torch.isfinite(got[seen]).any() and torch.isfinite(got[~seen]).all()
