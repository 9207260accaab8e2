"""Host parts of the packed operators: the prompt work list and the rotary
frequency rules.  No kernel is launched.  CPU only."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest


def _plan(lens, hq, hk, n_cta=148):
    from pse import _build, _native
    _build.build()
    lib = _native.load(require_cuda=False)
    host, n = np.asarray(lens, dtype=np.int32), ctypes.c_int64(0)
    args = (host.ctypes.data, len(lens), hq, hk, n_cta)
    assert lib.pse_prompt_plan(*args, None, 0, ctypes.addressof(n)) == 0
    out = np.full(n.value, -1, dtype=np.int32)
    assert lib.pse_prompt_plan(*args, out.ctypes.data, n.value, ctypes.addressof(n)) == 0
    head = (n_cta + 4) // 4 * 4
    return out[: n_cta + 1], out[head:].reshape(-1, 4), n.value


@pytest.mark.parametrize("lens,hq,hk", [([1], 1, 1), ([0, 300, 17, 0, 128], 32, 8), ([5000], 12, 12), ([3] * 500, 24, 3),
                                        ([700, 2], 130, 1), ([], 4, 2)])
def test_every_query_is_planned_once(lens, hq, hk):
    first, items, _ = _plan(lens, hq, hk)
    assert first[0] == 0 and first[-1] == len(items) and (np.diff(first) >= 0).all()
    per = 2 * max(1, 128 // (hq // hk))
    seen = np.zeros((sum(lens), hk), dtype=int)
    starts = dict()
    t = 0
    for n in lens:
        starts.setdefault(t, []).append(n)
        t += n
    for tok0, n, w0, h in items:
        assert n in starts[int(tok0)]
        seen[tok0 + w0: tok0 + min(n, w0 + per), h] += 1
    assert (seen == 1).all()


def test_work_is_dealt_evenly():
    lens = [8192, 5003, 700, 44, 44, 1]
    first, items, _ = _plan(lens, 32, 8)
    cost = [sum((min(n, w0 + 64) + 127) // 128 + 2 for _, n, w0, _ in items[a:b]) for a, b in zip(first, first[1:])]
    heaviest = (8192 + 127) // 128 + 2
    assert max(cost) - min(cost) <= heaviest and max(cost) <= sum(cost) / len(cost) * 1.05


def test_plan_refusals():
    from pse import _build, _native
    _build.build()
    lib = _native.load(require_cuda=False)
    n = ctypes.c_int64(0)
    lens = np.asarray([3, -1], dtype=np.int32)
    assert lib.pse_prompt_plan(lens.ctypes.data, 2, 4, 2, 148, None, 0, ctypes.addressof(n)) != 0
    lens = np.asarray([3, 1], dtype=np.int32)
    for hq, hk, cta in ((4, 3, 148), (0, 1, 148), (4, 2, 0)):
        assert lib.pse_prompt_plan(lens.ctypes.data, 2, hq, hk, cta, None, 0, ctypes.addressof(n)) != 0
    out = np.zeros(4, dtype=np.int32)
    assert lib.pse_prompt_plan(lens.ctypes.data, 2, 4, 2, 148, out.ctypes.data, 4, ctypes.addressof(n)) == 10002


def test_frequency_rules():
    from pse import rotary_frequencies
    plain, one = rotary_frequencies(64)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[31], 10000.0 ** (-62 / 64), rel_tol=1e-15)
    lin, _ = rotary_frequencies(64, scaling={"type": "linear", "factor": 4.0})
    assert all(math.isclose(a * 4, b, rel_tol=1e-15) for a, b in zip(lin, plain))
    # the base grows until the lowest frequency is divided by the factor; the highest stays
    ntk, _ = rotary_frequencies(64, scaling={"type": "ntk", "factor": 8.0})
    assert ntk[0] == 1.0 and math.isclose(ntk[31] * 8, plain[31], rel_tol=1e-12)
    bands, _ = rotary_frequencies(64, scaling={"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192})
    turns = [8192 * f / (2 * math.pi) for f in plain]
    for f, g, t in zip(plain, bands, turns):
        if t >= 4:
            assert g == f
        elif t <= 1:
            assert math.isclose(g * 8, f, rel_tol=1e-15)
        else:
            assert f / 8 < g < f
    yarn, factor = rotary_frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original": 4096})
    assert math.isclose(factor, 0.1 * math.log(16.0) + 1.0) and yarn[0] == plain[0]
    assert math.isclose(yarn[31] * 16, plain[31], rel_tol=1e-12)
    assert all(f / 16.000001 <= g <= f for f, g in zip(plain, yarn))
    _, factor = rotary_frequencies(64, scaling={"type": "yarn", "factor": 16.0, "original": 4096, "attention_factor": 1.0})
    assert factor == 1.0
    assert rotary_frequencies(0) == ([], 1.0)


@pytest.mark.parametrize("bad", [{"type": "x"}, {"type": "linear"}, {"type": "linear", "factor": 0},
                                 {"type": "bands", "factor": 8.0, "low": 4.0, "high": 1.0, "original": 8192},
                                 {"type": "yarn", "factor": 8.0}, {"type": "ntk", "factor": float("nan")}])
def test_frequency_refusals(bad):
    from pse import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(64, scaling=bad)


@pytest.mark.parametrize("factor,want", [(1.0, 1.0), (0.5, 1.0), (1e-6, 1.0), (2.0, 0.1 * math.log(2.0) + 1.0)])
def test_yarn_does_not_flatten_the_logits_of_shortened_contexts(factor, want):
    """The temperature belongs to contexts that grew; below a factor of 1 it stays 1."""
    from pse import rotary_frequencies
    f, got = rotary_frequencies(64, scaling={"type": "yarn", "factor": factor, "original": 4096})
    assert math.isclose(got, want, rel_tol=1e-15) and math.isclose(f[31] * factor, 10000.0 ** (-62 / 64), rel_tol=1e-12)
