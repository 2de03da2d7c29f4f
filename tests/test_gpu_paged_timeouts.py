"""Paged and prompt attention whose bounded waits give up: the call ends, says so, and the
next one is right.  The limit is lowered on the host until healthy waits run out."""
from __future__ import annotations

import contextlib

import pytest
import torch

from paged_ref import BF16, F16, F32, Pool
from test_gpu_paged import rand, run_paged
from test_gpu_prompt_attention import run_prompt

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def wait_limit(engine, cycles):
    from hf_llm_b200._lib import check, lib
    check(lib().b2q_set_wait_limit_cycles(engine.handle, cycles))
    try:
        yield
    finally:
        check(lib().b2q_set_wait_limit_cycles(engine.handle, 0))


def given_up(engine):
    """Whether a wait gave up since the last look (nothing else may have gone wrong)."""
    from hf_llm_b200._lib import ETIMEOUT, B2QError
    try:
        engine.check_device_error()
        return False
    except B2QError as e:
        assert e.status == ETIMEOUT, e
        return True


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,n", [(1, 1, 128, 8192), (16, 4, 128, 5000), (4, 1, 64, 12000), (4, 4, 64, 120)])
def test_a_prompt_call_that_gives_up_ends_and_the_next_one_is_right(engine, pkg, type_, heads, kv, dim, n):
    q, k, v = (rand((n, h, dim), s, type_) for h, s in ((heads, 1), (kv, 2), (kv, 3)))
    want = run_prompt(engine, heads, kv, dim, type_, [n], [n], q, k, v, 0.1)
    engine.check_device_error()
    for limit in (1, 300, 20000):
        with wait_limit(engine, limit):
            out = run_prompt(engine, heads, kv, dim, type_, [n], [n], q, k, v, 0.1)
        if not given_up(engine):
            assert n < 1000  # (the look at the last value tiles waits as long as the longest item takes)
            assert torch.equal(out, want)
        assert torch.equal(run_prompt(engine, heads, kv, dim, type_, [n], [n], q, k, v, 0.1), want)
        engine.check_device_error()


@pytest.mark.parametrize("lens,news", [([585], [1]), ([3000, 17, 900], [2, 1, 5])])
def test_a_paged_call_that_gives_up_ends_and_the_next_one_is_right(engine, pkg, lens, news):
    pool = Pool(8, 2, 128, 64, lens, news)
    pool.fill()
    pool.upload()
    q = rand((pool.rows, 8, 128), 1)
    want = run_paged(engine, pool, q, F32, F32, 0.1)
    engine.check_device_error()
    for limit in (1, 300):
        with wait_limit(engine, limit):
            out = run_paged(engine, pool, q, F32, F32, 0.1)
        if not given_up(engine):
            assert torch.equal(out, want)
        assert torch.equal(run_paged(engine, pool, q, F32, F32, 0.1), want)
        engine.check_device_error()
