"""Packed prompt attention over values that are not finite: they show in the rows that see
their key, and neither change another row nor hold up the call."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_ref import BF16, F16, TYPES
from test_gpu_paged_timeouts import wait_limit
from test_gpu_prompt_attention import pad, rand, run_prompt  # noqa: F401

pytestmark = pytest.mark.gpu


def expect(out, zeroed, v, heads, news, lens):
    """`zeroed`: the outputs with zeros for the bad values.  Where a row sees none in a
    column the bits are those; where it sees some, NaN if one is NaN or both signs are
    there, and that infinity (or NaN: its weight may have been rounded to 0) otherwise."""
    kv = v.shape[1]
    a = b = 0
    for n, l in zip(news, lens):
        x = v[b:b + l].float()
        up, down = (((x == s * float("inf")) | torch.isnan(x)).cumsum(0) > 0 for s in (1, -1))
        see = torch.arange(l - n, l)
        none = see < 0
        up, down = ((y[see.clamp(min=0)] & ~none[:, None, None]).repeat_interleave(heads // kv, 1) for y in (up, down))
        got, want = out[a:a + n].float().cpu(), zeroed[a:a + n].float().cpu()
        assert torch.equal(got[~up & ~down], want[~up & ~down])
        assert torch.isnan(got[up & down]).all()
        for hit, s in ((up & ~down, 1), (down & ~up, -1)):
            assert ((got[hit] == s * float("inf")) | torch.isnan(got[hit])).all()
        a, b = a + n, b + l


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,news,lens,share", [
    (4, 2, 64, [330, 60], [330, 60], 3e-4),
    (8, 2, 128, [100, 1, 257], [400, 300, 257], 3e-4),
    (2, 2, 128, [256, 255, 20], [700, 255, 10], 1e-3),   # 20 queries of 10 keys
    (6, 1, 64, [129], [1000], 0.02),
    (32, 8, 128, [500, 310, 64], [500, 900, 64], 1e-4),  # several items a CTA
    (1, 1, 128, [70], [70], 1.0),                        # nothing is finite
    # many items with one row tile between those with two
    (64, 8, 64, [1 + 7 * i % 41 for i in range(80)], [1 + 7 * i % 41 + 97 * i % 300 for i in range(80)], 1e-3),
])
def test_bad_values_anywhere(engine, pkg, type_, heads, kv, dim, news, lens, share):
    q, k, v = (rand((sum(x), h, dim), s, type_) for s, (x, h) in enumerate(((news, heads), (lens, kv), (lens, kv))))
    rng = np.random.default_rng(heads + dim)
    bad = torch.from_numpy(rng.random(v.shape) < share)
    zeros = torch.where(bad, torch.zeros_like(v), v)
    what = torch.from_numpy(rng.choice([np.inf, np.inf, -np.inf, np.nan], v.shape)).to(TYPES[type_])
    v = torch.where(bad, what, v)
    zeroed = run_prompt(engine, heads, kv, dim, type_, news, lens, q, k, zeros, 0.1)
    out = run_prompt(engine, heads, kv, dim, type_, news, lens, q, k, v, 0.1)
    expect(out, zeroed, v, heads, news, lens)
    engine.check_device_error()


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("at", [20000, 21000, 21999])
def test_a_bad_value_behind_a_long_prefix_holds_nothing_up(engine, pkg, type_, at):
    """2000 tokens behind 20000, two work items and more a CTA: within waits of 2e6 cycles."""
    heads, kv, dim, n, l = 32, 8, 128, 2000, 22000
    q, k, v = (rand((x, h, dim), s, type_) for s, (x, h) in enumerate(((n, heads), (l, kv), (l, kv))))
    v[at, 3, 17] = 0.0
    with wait_limit(engine, 2_000_000):
        zeroed = run_prompt(engine, heads, kv, dim, type_, [n], [l], q, k, v, 0.1)
        engine.check_device_error()
        for bad in (float("inf"), float("nan")):
            v[at, 3, 17] = bad
            out = run_prompt(engine, heads, kv, dim, type_, [n], [l], q, k, v, 0.1)
            engine.check_device_error()
            expect(out, zeroed, v, heads, [n], [l])


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_no_keys_in_the_call(engine, pkg, type_, dim):
    """n_kv = 0, with NULL keys and values: zeros."""
    q = rand((40, 4, dim), 1, type_)
    none = torch.empty(0, 2, dim, dtype=TYPES[type_])
    out = run_prompt(engine, 4, 2, dim, type_, [30, 0, 10], [0, 0, 0], q, none, none, 0.1)
    assert (out == 0).all()
    engine.check_device_error()
