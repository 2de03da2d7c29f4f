"""Rows of the paged attention that one call treats apart: the precision of a row
hangs on what that row sees, and rows without a valid position are left as they are."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, F32, TYPES, Pool
from test_gpu_paged import E_SCORE, e_prob, rand, run_paged, table  # noqa: F401

pytestmark = pytest.mark.gpu


def scale_tokens(pool, s, positions, factor, keys=False):
    """Multiplies the value (or key) scales of positions of sequence s by a power of two."""
    at = (8 if keys else 17) * pool.D
    for p in positions:
        blk = pool.pages[pool.table[s, p // pool.P], :, p % pool.P // 16]
        sc = blk[:, at:at + pool.D].copy().view(np.float16).reshape(pool.KV, 16, -1)
        new = (sc[:, p % 16].astype(np.float32) * factor).astype(np.float16)
        assert (new.astype(np.float32) == sc[:, p % 16].astype(np.float32) * factor).all()
        sc[:, p % 16] = new
        blk[:, at:at + pool.D] = sc.reshape(pool.KV, -1).view(np.uint8)


def value_scales(pool, s):
    """[len, KV]: the largest value scale of each token."""
    out = np.zeros((pool.lens[s], pool.KV))
    for p in range(pool.lens[s]):
        blk = pool.pages[pool.table[s, p // pool.P], :, p % pool.P // 16]
        sc = blk[:, 17 * pool.D:].copy().view(np.float16).reshape(pool.KV, 16, -1)
        out[p] = np.abs(sc[:, p % 16].astype(np.float64)).max(-1)
    return out


def check_rows(out, pool, ks, vs, q, scale, q_type, out_type):
    """Each row against f64 by itself.  A probability times its value's scale enters as
    f16, one part or two, and the largest such product that the row has is 2^6 or above: a
    term is off by 2^-25 (half of f16's smallest step) beside its relative error, so by 2^-31
    of that product, times |code - 8| <= 8.  (1.02: the kernel's own probabilities.)"""
    G, a = pool.H // pool.KV, 0
    for s, n in enumerate(pool.news):
        l, top = pool.lens[s], value_scales(pool, s)
        for i in range(n):
            see = l - n + i + 1
            x = q[a + i].double()
            for h in range(pool.H):
                w = torch.from_numpy(ks[s][:see, h // G]) @ x[h] * scale
                m = float((torch.softmax(w, 0) * torch.from_numpy(top[:see, h // G])).max())
                want, bound = R.attend(x[None, h:h + 1], [ks[s][:see, h // G:h // G + 1]], [vs[s][:see, h // G:h // G + 1]], [1], scale,
                                       TYPES[out_type], E_SCORE, e_prob(out_type), 1.02 * 2.0 ** -28 * m)
                R.check_close(out[a + i:a + i + 1, h:h + 1], want, bound)
        a += n


@pytest.mark.parametrize("heads,kv,dim,lens,news,q_type,out_type", [
    (8, 2, 128, [300, 40], [5, 3], F32, F32),
    (16, 2, 64, [70, 33], [4, 2], F16, F32),     # 16 rows to an item
    (8, 1, 128, [130], [3], BF16, BF16),
    (4, 4, 64, [17, 64], [2, 5], F32, F16),
])
def test_a_row_keeps_its_bits_beside_values_it_does_not_see(engine, pkg, heads, kv, dim, lens, news, q_type, out_type):
    """The last new token's values are 2^27 times the others'."""
    pool = Pool(heads, kv, dim, 16, lens, news, seed=2)
    ks, vs = pool.fill()
    for s, l in enumerate(lens):
        scale_tokens(pool, s, range(l - 1), 2.0 ** -10)
        scale_tokens(pool, s, [l - 1], 2.0 ** 17)
        vs[s][:l - 1] *= 2.0 ** -10
        vs[s][l - 1] *= 2.0 ** 17
    q = rand((pool.rows, heads, dim), 5, q_type)
    out = run_paged(engine, pool.upload(), q, q_type, out_type, dim ** -0.5)
    check_rows(out, pool, ks, vs, q, dim ** -0.5, q_type, out_type)
    engine.check_device_error()


@pytest.mark.parametrize("q_type,out_type", [(F32, F32), (F16, F16)])
@pytest.mark.parametrize("at", [0, 7, 100, 298])
def test_large_values_without_weight(engine, pkg, q_type, out_type, at):
    """One token with values 2^27 times the others' and a probability below 2^-50."""
    pool = Pool(8, 2, 128, 16, [300], [1], seed=2)
    ks, vs = pool.fill()
    scale_tokens(pool, 0, [p for p in range(300) if p != at], 2.0 ** -10)
    scale_tokens(pool, 0, [at], 2.0 ** 17)
    scale_tokens(pool, 0, [at], 8.0, keys=True)
    f = np.where(np.arange(300) == at, 2.0 ** 17, 2.0 ** -10)[:, None, None]
    vs[0] *= f
    ks[0][at] *= 8.0
    # queries that point away from that token's key
    q = rand((1, 8, 128), 5).double()
    for h in range(8):
        k = torch.from_numpy(ks[0][at, h // 4])
        q[0, h] -= 6.0 * k / k.norm() + (q[0, h] @ k) * k / (k @ k)
    q = q.to(TYPES[q_type])
    w = torch.einsum("hd,hd->h", q[0].double(), torch.from_numpy(ks[0][at]).repeat_interleave(4, 0)) * 128 ** -0.5
    assert (w < -36).all()  # e^-36 < 2^-51
    out = run_paged(engine, pool.upload(), q, q_type, out_type, 128 ** -0.5)
    check_rows(out, pool, ks, vs, q, 128 ** -0.5, q_type, out_type)


def rows_left(engine, pool, ks, vs, q, q_type, claimed, cap, scale=0.125):
    """Runs with kv_len = claimed: rows with a position in [0, cap) attend the keys that the
    table has, the others keep what they held."""
    from hf_llm_b200._lib import B2QError, EINVAL
    n, real = pool.news[0], pool.lens[0]
    pool.dev["kv_len"][0] = claimed
    out = run_paged(engine, pool, q, q_type, q_type, scale)
    with pytest.raises(B2QError) as e:
        engine.check_device_error()
    assert e.value.status == EINVAL
    for i in range(n):
        pos = claimed - n + i
        if 0 <= pos < cap:
            see = min(pos + 1, real)
            want, bound = R.attend(q[i:i + 1].double(), [ks[0][:see]], [vs[0][:see]], [1], scale, TYPES[q_type], E_SCORE, e_prob(q_type),
                                   2.0 ** -28 * pool.largest_scale())
            R.check_close(out[i:i + 1], want, bound)
        else:
            assert (out[i] == 7.0).all(), (i, pos)
    want, bound = R.attend(q[n:pool.T].double(), ks[1:], vs[1:], pool.news[1:], scale, TYPES[q_type], E_SCORE, e_prob(q_type),
                           2.0 ** -28 * pool.largest_scale())
    R.check_close(out[n:pool.T], want, bound)


@pytest.mark.parametrize("q_type", [F32, F16])
@pytest.mark.parametrize("pages,page", [(4, 16), (16, 256)])  # a cluster an item; one line, joined by a second launch
def test_rows_without_a_position_are_left_as_they_are(engine, pkg, q_type, pages, page):
    cap = pages * page
    pool = Pool(8, 1, 64, page, [cap, 20], [4, 2], max_pages=pages)
    ks, vs = pool.fill()
    pool.upload()
    q = rand((pool.rows, 8, 64), 5, q_type)
    # the sequence's keys are those of the table, whatever kv_len claims
    for claimed in (cap + 1, cap + 3, cap + 4, cap + 100, 2 ** 31 - 1, 3, 1, 0, -1, -2 ** 31):
        rows_left(engine, pool, ks, vs, q, q_type, claimed, cap)


def offsets_reported(engine, f):
    from hf_llm_b200._lib import B2QError, EINVAL
    f()
    torch.cuda.synchronize()
    with pytest.raises(B2QError) as e:
        engine.check_device_error()
    assert e.value.status == EINVAL
    engine.check_device_error()


@pytest.mark.parametrize("seqs", [2, 150, 1500])
def test_offsets_that_decrease_are_reported(engine, pkg, seqs):
    """By each of the four calls, also where no row of the call falls into the
    sequence that they belong to."""
    from hf_llm_b200 import paged
    start = [0] * (seqs - 1) + [3, 2]
    H, KV, D, st = 4, 2, 64, 1
    cfg = paged.kv_config(H, KV, D, R.Q4_0, 16, seqs, 1)
    qs = torch.tensor(start, dtype=torch.int32).cuda()
    lens = torch.full((seqs,), 16, dtype=torch.int32).cuda()
    tab = torch.arange(seqs, dtype=torch.int32).cuda()
    pages = torch.zeros(seqs * paged.page_bytes(cfg), dtype=torch.uint8, device="cuda")
    b = paged.kv_batch(seqs, 4, 3, qs.data_ptr(), lens.data_ptr(), tab.data_ptr())
    q, k, v = (rand((4, h, D), i, F16).cuda() for i, h in enumerate((H, KV, KV)))
    out = torch.empty_like(q)
    work = torch.empty(engine.attn_paged_work_bytes(cfg, b), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    engine.check_device_error()
    offsets_reported(engine, lambda: engine.kv_append_dev(cfg, b, None, F16, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D,
                                                          pages.data_ptr(), out.data_ptr(), F16, st))
    offsets_reported(engine, lambda: engine.kv_gather_dev(cfg, b, pages.data_ptr(), k.data_ptr(), v.data_ptr(), F16, st))
    offsets_reported(engine, lambda: engine.attn_paged_dev(cfg, b, q.data_ptr(), F16, H * D, pages.data_ptr(), 0.1, out.data_ptr(), F16,
                                                           work.data_ptr(), work.numel(), st))
    ks = torch.tensor([0] * seqs + [4], dtype=torch.int32).cuda()
    p = paged.prompt(H, KV, D, F16, seqs, 4, 4, 3, qs.data_ptr(), ks.data_ptr())
    offsets_reported(engine, lambda: engine.attn_prompt_dev(p, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D, 0.1,
                                                            out.data_ptr(), st))


def test_scores_of_zero_under_a_large_scale(engine, pkg):
    """Keys of zeros under queries and a scale whose product passes f32's range: all
    scores are 0, and the output is the values' mean."""
    pool = Pool(4, 2, 64, 16, [50], [1])
    ks, vs = pool.fill()
    scale_tokens(pool, 0, range(50), 0.0, keys=True)
    q = torch.full((1, 4, 64), 1e20)
    out = run_paged(engine, pool.upload(), q, F32, F32, 1e30)
    mean = torch.from_numpy(vs[0].mean(0)).repeat_interleave(2, 0)[None]
    # two parts of each probability times scale, 2^-21, and eight f32 roundings on the way out
    R.check_close(out, mean, torch.full_like(mean, 2.0 ** -20 * float(np.abs(vs[0]).max())))
    engine.check_device_error()
