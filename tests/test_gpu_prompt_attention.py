"""Packed causal attention on a B200 (b2q_attn_prompt_dev) against attention
in f64, within bounds derived from its roundings (paged_ref.attend)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, TYPES

pytestmark = pytest.mark.gpu


def rand(shape, seed, type_, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(TYPES[type_])


PAD = 0


@pytest.fixture(autouse=True, params=[0, 20000], ids=["few rows", "many rows"])
def pad(request):
    """Rows behind the last sequence: with many of them the call takes two row
    tiles at a time instead of one in two halves."""
    global PAD
    PAD = request.param
    yield
    PAD = 0


def run_prompt(engine, heads, kv, dim, type_, news, lens, q, k, v, scale, max_new=None, strides=None, n_q=None, stream=None, out=None):
    from hf_llm_b200 import paged
    qs = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32).cuda()
    ks = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    q, k, v = (x if x.is_cuda else x.cuda() for x in (q, k, v))
    rows = q.shape[0]
    if PAD and out is None and strides is None:
        q = torch.cat([q, torch.full((PAD,) + tuple(q.shape[1:]), float("nan"), dtype=q.dtype, device="cuda")])
    n_q = q.shape[0] if n_q is None else n_q
    if out is None:
        out = torch.full((q.shape[0], heads, dim), 7.0, dtype=TYPES[type_], device="cuda")
    st = strides or (heads * dim, kv * dim, kv * dim)
    p = paged.prompt(heads, kv, dim, type_, len(news), n_q, k.shape[0], max(news) if max_new is None else max_new,
                     qs.data_ptr(), ks.data_ptr())
    torch.cuda.synchronize()
    engine.attn_prompt_dev(p, q.data_ptr(), st[0], k.data_ptr(), st[1], v.data_ptr(), st[2], scale, out.data_ptr(),
                           stream or torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    assert (out[rows:] == 7.0).all()
    return out[:rows]


def tiny(type_, v):
    """A probability, the largest at 2^7 or above, is off by at most half of f16's
    smallest step, 2^-25, as well: 2^-32 of the largest value to each key's
    term, the sum of the probabilities being at least 1.  (bf16 has f32's range.)"""
    return 2.0 ** -32 * float(v.float().abs().max()) if type_ == F16 and v.numel() else 0.0


def e_prob(type_):
    return R.half_eps(TYPES[type_])


def check(engine, heads, kv, dim, type_, news, lens, scale=None, spread=1.0, seed=0, extra=0, **kw):
    T, L = sum(news), sum(lens)
    q = rand((T + extra, heads, dim), seed + 1, type_, spread)
    k, v = rand((L + extra, kv, dim), seed + 2, type_), rand((L + extra, kv, dim), seed + 3, type_)
    if extra:  # rows that no sequence has
        k[L:], v[L:] = float("nan"), float("nan")
    scale = scale or dim ** -0.5
    out = run_prompt(engine, heads, kv, dim, type_, news, lens, q, k, v, scale, **kw)
    at = np.concatenate([[0], np.cumsum(lens)])
    rows = [[x[a:b].double().numpy() for a, b in zip(at[:-1], at[1:])] for x in (k, v)]
    # products of 16-bit values in f32 sums: 2^-19 of their magnitudes; the
    # probabilities are rounded to the type, relative to a maximum that may lag
    want, bound = R.attend(q[:T].double(), rows[0], rows[1], news, scale, TYPES[type_], 2.0 ** -19, e_prob(type_),
                           tiny(type_, v[:L]))
    if T:
        R.check_close(out[:T], want, bound)
    assert (out[T:] == 7.0).all()  # rows behind the last sequence
    engine.check_device_error()
    return out


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,news,lens", [
    (1, 1, 64, [1], [1]),
    (8, 2, 128, [1, 2, 3], [1, 2, 3]),
    (4, 1, 128, [127, 128, 129], [127, 128, 129]),
    (8, 8, 64, [255, 256, 257], [255, 256, 257]),
    (6, 2, 128, [300], [300]),
    (9, 3, 64, [65, 0, 130], [65, 0, 130]),            # a sequence without tokens
    (8, 2, 128, [1, 1, 1], [700, 129, 128]),           # the next token behind a prefix
    (4, 2, 64, [50, 200, 7], [300, 201, 1024]),
    (2, 1, 128, [130, 10], [130 + 255, 10 + 120]),
    (16, 1, 128, [33, 64, 100, 17], [33, 64, 100, 17]),
    (4, 2, 64, [3, 5], [0, 0]),                        # no keys at all
    (3, 3, 64, [20, 9], [10, 9]),                      # more queries than keys: the first ones have none
    (2, 2, 128, [700], [1500]),
])
def test_packed_prompts(engine, pkg, type_, heads, kv, dim, news, lens):
    out = check(engine, heads, kv, dim, type_, news, lens, extra=3)
    assert torch.equal(out, check(engine, heads, kv, dim, type_, news, lens, extra=3, max_new=0))  # the hint
    if sum(lens) == 0:
        assert (out[:8] == 0).all()
    if news == [20, 9]:
        assert (out[:10] == 0).all()


@pytest.mark.parametrize("spread,scale", [(20.0, 0.09), (1e-3, 0.09), (8.0, 1.0), (1.0, 1e-4)])
@pytest.mark.parametrize("type_", [F16, BF16])
def test_peaked_and_flat(engine, pkg, type_, spread, scale):
    check(engine, 4, 2, 128, type_, [190, 300], [300, 300], scale=scale, spread=spread)
    check(engine, 4, 2, 64, type_, [300], [300], scale=scale, spread=spread)


def test_growing_scores(engine, pkg):
    """Keys whose scores grow along the sequence: the running maximum moves in
    every tile, by a little and by a lot."""
    for step in (0.02, 0.5, 3.0):
        L, D = 700, 128
        k = torch.zeros(L, 1, D)
        k[:, 0, 0] = torch.arange(L) * step / 16
        k[:, 0, 1:] = rand((L, D - 1), 3, F16).float() * 0.1
        q = rand((L, 2, D), 4, F16).float() * 0.1
        q[:, :, 0] = 16.0
        q, k, v = q.half(), k.half(), rand((L, 1, D), 5, F16)
        out = run_prompt(engine, 2, 1, D, F16, [L], [L], q, k, v, 1.0)
        want, bound = R.attend(q.double(), [k.double().numpy()], [v.double().numpy()], [L], 1.0, torch.float16, 2.0 ** -19, e_prob(F16), tiny(F16, v))
        # scores up to 16 * 131: the exponent's argument is rounded at that size
        R.check_close(out, want, bound + 4 * 2.0 ** -24 * 16 * 131 * 1.45 * 4.0)


def test_strided_rows_of_one_projection(engine, pkg):
    H, KV, D, n = 4, 2, 64, 150
    row = rand((n, (H + 2 * KV) * D), 2, BF16).cuda()
    q, k, v = row[:, :H * D], row[:, H * D:(H + KV) * D], row[:, (H + KV) * D:]
    out = torch.full((n, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    run_prompt(engine, H, KV, D, BF16, [100, 50], [100, 50], q, k, v, 0.125, strides=((H + 2 * KV) * D,) * 3, out=out)
    same = run_prompt(engine, H, KV, D, BF16, [100, 50], [100, 50], q.contiguous(), k.contiguous(), v.contiguous(), 0.125)
    assert torch.equal(out, same.view_as(out))


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(engine, pkg, type_, dim, bad):
    """A bad value row at key 200 of the first sequence: queries before it, and
    the other sequence, get the bits they get without it."""
    news, lens = [330, 60], [330, 60]
    q, k, v = (rand((390, h, dim), s, type_) for h, s in ((4, 1), (2, 2), (2, 3)))
    ok = run_prompt(engine, 4, 2, dim, type_, news, lens, q, k, v, 0.1)
    w = v.clone()
    w[200, 0, 5] = bad
    out = run_prompt(engine, 4, 2, dim, type_, news, lens, q, k, w, 0.1)
    assert torch.equal(out[330:], ok[330:])
    assert torch.equal(out[:, 2:], ok[:, 2:])  # the other K/V head
    want, bound = R.attend(q[:200].double(), [k[:200].double().numpy()], [v[:200].double().numpy()], [200], 0.1, TYPES[type_],
                           2.0 ** -19, e_prob(type_), tiny(type_, v))
    R.check_close(out[:200], want, bound)
    hit = out[200:330, :2, 5].float()
    assert (~torch.isfinite(hit)).all()
    if bad == bad:
        assert ((hit == bad) | torch.isnan(hit)).all()
    rest = torch.cat([out[200:330, :2, :5], out[200:330, :2, 6:]], -1)
    assert torch.isfinite(rest).all()
    engine.check_device_error()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_keys_and_queries_that_are_not_finite(engine, pkg, bad):
    q, k, v = (rand((390, h, 128), s, F16) for h, s in ((4, 1), (2, 2), (2, 3)))
    ok = run_prompt(engine, 4, 2, 128, F16, [330, 60], [330, 60], q, k, v, 0.1)
    k2 = k.clone()
    k2[200, 0, 5] = bad
    out = run_prompt(engine, 4, 2, 128, F16, [330, 60], [330, 60], q, k2, v, 0.1)
    assert torch.equal(out[330:], ok[330:]) and torch.equal(out[:200], ok[:200]) and torch.equal(out[:, 2:], ok[:, 2:])
    for at in range(200, 216):  # whatever the key's column, the rows whose score is NaN or +inf show it
        k2 = k.clone()
        k2[at, 0, 5] = bad
        got = run_prompt(engine, 4, 2, 128, F16, [330, 60], [330, 60], q, k2, v, 0.1)
        score = q[at:330, :2, 5].float() * bad
        hit = torch.isnan(score) | (score == float("inf"))
        assert torch.equal(torch.isnan(got[at:330, :2].cpu()).all(-1), hit) and torch.isfinite(got[at:330, :2].cpu()[~hit]).all()
    q2 = q.clone()
    q2[150, 1, 3] = float("nan")
    out = run_prompt(engine, 4, 2, 128, F16, [330, 60], [330, 60], q2, k, v, 0.1)
    assert torch.isnan(out[150, 1]).all()
    out[150, 1] = ok[150, 1]
    assert torch.equal(out, ok)


def test_scores_of_minus_infinity_beside_values_that_are_not_finite(engine, pkg):
    """Key 0 scores -inf where the query's dim 5 is positive: no weight, also in
    rows that are computed again for an infinite value behind them."""
    q, k, v = (rand((330, h, 64), s, F16) for h, s in ((4, 1), (2, 2), (2, 3)))
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    k[0, :, 5] = -float("inf")
    v[200, 0, 7] = float("inf")
    out = run_prompt(engine, 4, 2, 64, F16, [330], [330], q, k, v, 0.1)
    # the same without key 0, which the first query then has nothing of
    want, bound = R.attend(q[1:200].double(), [k[1:200].double().numpy()], [v[1:200].double().numpy()], [199], 0.1, TYPES[F16],
                           2.0 ** -19, e_prob(F16), tiny(F16, v[:200]))
    R.check_close(out[1:200], want, bound)
    assert torch.isinf(out[200:, :2, 7]).all()


def test_offsets_out_of_range_are_reported(engine, pkg):
    from hf_llm_b200 import paged
    from hf_llm_b200._lib import B2QError, EINVAL
    q, k, v = (rand((64, h, 64), s, F16).cuda() for h, s in ((4, 1), (2, 2), (2, 3)))
    for qs, ks in (([0, 40, 64], [0, 40, 100]), ([0, 40, 64], [0, -1, 64]), ([0, 40, 64], [30, 10, 64]), ([0, 40, 100], [0, 40, 64]),
                   ([0, 2 ** 31 - 1, 64], [0, 40, 64]), ([-5, 40, 64], [0, 40, 64]),
                   ([0, 40, 64], [-2 ** 31, 2 ** 31 - 1, 64])):
        out = torch.full((64, 4, 64), 7.0, dtype=torch.float16, device="cuda")
        a, b = (torch.tensor(x, dtype=torch.int32).cuda() for x in (qs, ks))
        p = paged.prompt(4, 2, 64, F16, 2, 64, 64, 0, a.data_ptr(), b.data_ptr())
        torch.cuda.synchronize()
        engine.attn_prompt_dev(p, q.data_ptr(), 256, k.data_ptr(), 128, v.data_ptr(), 128, 0.1, out.data_ptr(), 1)
        torch.cuda.synchronize()
        assert torch.isfinite(out).all()
        with pytest.raises(B2QError) as e:
            engine.check_device_error()
        assert e.value.status == EINVAL, (qs, ks)


def test_captured_and_replayed_with_other_lengths(engine, pkg):
    """One capture, replayed after the device offsets changed."""
    from hf_llm_b200 import paged
    q, k, v = (rand((300, h, 64), s, BF16).cuda() for h, s in ((4, 1), (2, 2), (2, 3)))
    out = torch.empty(300, 4, 64, dtype=torch.bfloat16, device="cuda")
    offs = torch.tensor([0, 100, 300], dtype=torch.int32).cuda()
    p = paged.prompt(4, 2, 64, BF16, 2, 300, 300, 300, offs.data_ptr(), offs.data_ptr())
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        engine.attn_prompt_dev(p, q.data_ptr(), 256, k.data_ptr(), 128, v.data_ptr(), 128, 0.125, out.data_ptr(), s.cuda_stream)
    for mid, end in ((100, 300), (299, 300), (0, 17), (140, 260)):
        offs.copy_(torch.tensor([0, mid, end], dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        want = run_prompt(engine, 4, 2, 64, BF16, [mid, end - mid], [mid, end - mid], q, k, v, 0.125, out=torch.full_like(out, 7.0))
        assert torch.equal(out, want)


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,news,lens", [
    (2, 2, [256, 255, 1], [2300, 2049, 2304]),   # three tiles with the causal edge behind many whole ones
    (1, 1, [1100], [1100]),
    (4, 1, [200, 190], [1500, 200]),
])
def test_long_prefixes_and_many_tiles(engine, pkg, type_, dim, heads, kv, news, lens):
    """Key tiles go round the ring several times, and the last tiles wait for
    the look at their values: again and again the same bits."""
    out = check(engine, heads, kv, dim, type_, news, lens, extra=130)
    for _ in range(5):
        assert torch.equal(out, check(engine, heads, kv, dim, type_, news, lens, extra=130))
