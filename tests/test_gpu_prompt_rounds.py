"""Packed prompt attention where a CTA goes from item to item: more work items than SMs,
several key tiles each, items of one and of two row tiles in turn."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, TYPES
from test_gpu_prompt_attention import check, e_prob, rand, run_prompt, tiny

pytestmark = pytest.mark.gpu


def ragged(seed, n, lo, hi, prefix):
    rng = np.random.default_rng(seed)
    news = [int(x) for x in rng.integers(lo, hi + 1, n)]
    return news, [a + int(x) * int(y) for a, x, y in zip(news, rng.integers(0, prefix + 1, n), rng.integers(0, 2, n))]


def real_items(heads, kv, news, lens):
    """(row tiles, key tiles) of the items that have rows, as the two-row-tile form cuts them."""
    tpt = 128 // min(heads // kv, 64)
    return [(2 if at + tpt < n else 1, -(-(min(n, at + 2 * tpt) + l - n) // 128))
            for n, l in zip(news, lens) for at in range(0, n, 2 * tpt) for _ in range(kv)]


@pytest.mark.parametrize("type_", [F16, BF16])
@pytest.mark.parametrize("heads,kv,dim,n,lo,hi,prefix", [
    (32, 8, 128, 6, 300, 900, 0),
    (32, 8, 64, 6, 300, 900, 500),
    (8, 8, 128, 12, 100, 600, 700),
    (12, 4, 64, 9, 150, 1100, 300),     # 42 tokens to a row tile
    (64, 8, 128, 40, 1, 40, 600),       # short rows behind long prefixes: most items have one row tile
])
def test_items_behind_one_another(engine, pkg, type_, heads, kv, dim, n, lo, hi, prefix):
    news, lens = ragged(heads + dim + n, n, lo, hi, prefix)
    items = real_items(heads, kv, news, lens)
    assert len(items) > 148 and {a for a, _ in items} == {1, 2} and max(b for _, b in items) >= 5
    out = check(engine, heads, kv, dim, type_, news, lens, extra=3)
    # (check()'s inputs) the same bits again and again
    T, L = sum(news), sum(lens)
    q, k, v = rand((T + 3, heads, dim), 1, type_), rand((L + 3, kv, dim), 2, type_), rand((L + 3, kv, dim), 3, type_)
    k[L:], v[L:] = float("nan"), float("nan")
    for _ in range(5):
        assert torch.equal(out, run_prompt(engine, heads, kv, dim, type_, news, lens, q, k, v, dim ** -0.5))


def test_one_head_apart_many_heads_together(engine, pkg):
    """The same rows with the heads one K/V head at a time (few items: one a CTA) and
    together (several a CTA), both against f64."""
    news, lens = [400, 37, 290], [400, 500, 290]
    H, KV, D = 64, 16, 128
    q, k, v = (rand((sum(x), h, D), s, BF16) for s, (x, h) in enumerate(((news, H), (lens, KV), (lens, KV))))
    all_ = run_prompt(engine, H, KV, D, BF16, news, lens, q, k, v, 0.09)
    at = np.concatenate([[0], np.cumsum(lens)])
    for kvh in (0, 7, 15):
        one = [x.contiguous() for x in (q[:, 4 * kvh:4 * kvh + 4], k[:, kvh:kvh + 1], v[:, kvh:kvh + 1])]
        rows = [[x[a:b].double().numpy() for a, b in zip(at[:-1], at[1:])] for x in one[1:]]
        want, bound = R.attend(one[0].double(), rows[0], rows[1], news, 0.09, TYPES[BF16], 2.0 ** -19, e_prob(BF16), tiny(BF16, v))
        R.check_close(run_prompt(engine, 4, 1, D, BF16, news, lens, *one, 0.09), want, bound)
        R.check_close(all_[:, 4 * kvh:4 * kvh + 4], want, bound)


@pytest.mark.parametrize("rows", [0, 20000], ids=["halves", "pairs"])
@pytest.mark.parametrize("dim", [64, 128])
def test_strided_captured_and_replayed(engine, pkg, dim, rows):
    """q | k | v rows of one projection, captured once and replayed with other lengths, in
    both forms of the call: the bits of contiguous calls made one by one."""
    from hf_llm_b200 import paged
    H, KV, n = 8, 2, 700
    T = n + rows
    W = (H + 2 * KV) * dim
    x = torch.full((T, W), float("nan"), dtype=torch.float16, device="cuda")
    x[:n] = rand((n, W), 3, F16).cuda()
    q, k, v = (x[:, a * dim:b * dim] for a, b in ((0, H), (H, H + KV), (H + KV, H + 2 * KV)))
    offs = torch.tensor([0, 100, 700], dtype=torch.int32).cuda()
    out = torch.full((T, H, dim), 7.0, dtype=torch.float16, device="cuda")
    p = paged.prompt(H, KV, dim, F16, 2, T, n, n, offs.data_ptr(), offs.data_ptr())
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        engine.attn_prompt_dev(p, q.data_ptr(), W, k.data_ptr(), W, v.data_ptr(), W, 0.125, out.data_ptr(), s.cuda_stream)
    cq, ck, cv = q.contiguous(), k[:n].contiguous(), v[:n].contiguous()
    for mid, end in ((100, 700), (699, 700), (0, 17), (333, 500)):
        offs.copy_(torch.tensor([0, mid, end], dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        one = torch.full_like(out, 7.0)
        run_prompt(engine, H, KV, dim, F16, [mid, end - mid], [mid, end - mid], cq, ck, cv, 0.125, out=one)
        assert torch.equal(out, one) and (out[end:] == 7.0).all()
    engine.check_device_error()


def test_two_large_calls_at_once(engine, pkg):
    from hf_llm_b200 import paged
    H, KV, D = 32, 8, 128
    news, _ = ragged(3, 7, 200, 700, 0)
    T = sum(news)
    start = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32).cuda()
    p = paged.prompt(H, KV, D, BF16, 7, T, T, 0, start.data_ptr(), start.data_ptr())
    x = [[rand((T, h, D), 10 * i + j, BF16).cuda() for j, h in enumerate((H, KV, KV))] for i in range(2)]

    def call(i, out, st):
        q, k, v = x[i]
        engine.attn_prompt_dev(p, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D, 0.09, out.data_ptr(), st)

    want = [torch.empty_like(x[i][0]) for i in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        call(i, want[i], 1)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(x[i][0]) for _ in range(5)] for i in range(2)]
    torch.cuda.synchronize()
    for n in range(5):
        for i in range(2):
            call(i, got[i][n], streams[i].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    engine.check_device_error()


def test_bad_offsets_leave_other_sequences_whole(engine, pkg):
    """One sequence's keys out of range among many items: reported, its rows left, the others'
    as without it."""
    from hf_llm_b200._lib import B2QError, EINVAL
    from hf_llm_b200 import paged
    H, KV, D, news = 32, 8, 64, [300, 260, 410, 333]
    T = sum(news)
    q, k, v = (rand((T, h, D), i, F16).cuda() for i, h in enumerate((H, KV, KV)))
    qs = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    outs = []
    for last in (T, T + 1):
        ks = qs.copy()
        ks[-1] = last
        a, b = torch.from_numpy(qs).cuda(), torch.from_numpy(ks).cuda()
        out = torch.full((T, H, D), 7.0, dtype=torch.float16, device="cuda")
        p = paged.prompt(H, KV, D, F16, 4, T, T, 0, a.data_ptr(), b.data_ptr())
        torch.cuda.synchronize()
        engine.attn_prompt_dev(p, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D, 0.125, out.data_ptr(), 1)
        torch.cuda.synchronize()
        outs.append(out)
        if last == T:
            engine.check_device_error()
        else:
            with pytest.raises(B2QError) as e:
                engine.check_device_error()
            assert e.value.status == EINVAL
    assert torch.equal(outs[0][:qs[3]], outs[1][:qs[3]]) and (outs[1][qs[3]:] == 7.0).all()
