"""The operators of the paged K/V cache together, as a host that serves several
requests calls them, on a B200: projections by the grouped product, append,
read-back, packed prompt attention, then tokens one by one and a drafted run; and
each of them at batches, heads and addresses beyond the ordinary."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, F32, Pool, TYPES
from test_gpu_paged import E_SCORE, check_paged, e_prob, expected_pages, rand, run_append, run_paged, stream, table, tiny  # noqa: F401
from test_gpu_prompt_attention import check as check_prompt
from test_gpu_prompt_attention import e_prob as e_prob_prompt, tiny as tiny_prompt

pytestmark = pytest.mark.gpu

Q8_0 = 8


class Layer:
    """One attention layer's cache, kept as a host does, beside a plain model of
    it: `hist` holds each sequence's f64 keys and values as the cache has them."""

    def __init__(self, engine, H, KV, D, E, page, n_seqs, room, seed):
        from hf_llm_b200 import paged
        self.engine, self.paged = engine, paged
        self.H, self.KV, self.D, self.E, self.P, self.n = H, KV, D, E, page, n_seqs
        rng = np.random.default_rng(seed)
        self.w = []
        for n in (H * D, KV * D, KV * D):
            code = rng.integers(-127, 128, (n, E // 32, 32)).astype(np.int8)
            scale = np.full((n, E // 32, 1), 1 / (73 * np.sqrt(E)), np.float16)  # weights of about 1 / sqrt(E)
            raw = np.concatenate([scale.view(np.uint8).reshape(n, E // 32, 2), code.view(np.uint8)], -1)
            w = (code * scale.astype(np.float64)).reshape(n, E)
            self.w.append((w, engine.try_upload_weight(raw.reshape(-1), Q8_0, n, E)))
        mp = (room + page - 1) // page
        perm = rng.permutation(n_seqs * mp).astype(np.int32).reshape(n_seqs, mp)
        self.cfg = paged.kv_config(H, KV, D, R.Q4_0, page, n_seqs * mp, mp + R.MORE_PAGES)
        self.table = torch.from_numpy(np.pad(perm, ((0, 0), (0, R.MORE_PAGES)), constant_values=-7)).cuda()
        self.pages = torch.full((n_seqs * mp * paged.page_bytes(self.cfg),), 0xff, dtype=torch.uint8, device="cuda")
        self.cos, self.sin = R.rope_tables(room, D)
        self.dev_tables = torch.from_numpy(self.cos).cuda(), torch.from_numpy(self.sin).cuda()
        self.rope = paged.rope(D, room, *(x.data_ptr() for x in self.dev_tables))
        self.lens = [0] * n_seqs
        self.hist = [[np.zeros((0, KV, D)), np.zeros((0, KV, D))] for _ in range(n_seqs)]

    def close(self):
        for _, b in self.w:
            b.free()

    def project(self, x):
        T = len(x)
        ns = [w.shape[0] for w, _ in self.w]
        y = torch.empty(T * sum(ns), device="cuda")
        torch.cuda.synchronize()
        self.engine.matmul_group_dev([(b, n) for n, (_, b) in zip(ns, self.w)], x.data_ptr(), y.data_ptr(), T, self.E, stream())
        torch.cuda.synchronize()
        out, at = [], 0
        for n, (w, _) in zip(ns, self.w):
            part = y[at:at + T * n].view(T, n)
            want = x.cpu().double().numpy() @ w.T
            err = np.linalg.norm(part.cpu().double().numpy() - want) / np.linalg.norm(want)
            assert err < 1e-2  # (the product has tests of its own)
            out.append(part)
            at += T * n
        return out

    def step(self, news, x, prompt_type=None):
        """Appends `news` tokens a sequence and attends them; each output against f64."""
        e, H, KV, D = self.engine, self.H, self.KV, self.D
        T = sum(news)
        q, k, v = self.project(x)
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.lens = [l + n for l, n in zip(self.lens, news)]
        d_start, d_len = torch.from_numpy(starts).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        batch = self.paged.kv_batch(self.n, T, max(news), d_start.data_ptr(), d_len.data_ptr(), self.table.data_ptr())
        t_out = F32 if prompt_type is None else prompt_type
        qr = torch.empty(T, H, D, dtype=TYPES[t_out], device="cuda")
        out = torch.full((T, H, D), 7.0, dtype=TYPES[t_out], device="cuda")
        torch.cuda.synchronize()
        e.kv_append_dev(self.cfg, batch, self.rope, F32, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D,
                        self.pages.data_ptr(), qr.data_ptr(), t_out, stream())
        if prompt_type is None:
            work = torch.empty(e.attn_paged_work_bytes(self.cfg, batch), dtype=torch.uint8, device="cuda")
            e.attn_paged_dev(self.cfg, batch, qr.data_ptr(), F32, H * D, self.pages.data_ptr(), D ** -0.5, out.data_ptr(), F32,
                             work.data_ptr(), work.numel(), stream())
        else:  # every cached token is read back for the prompt's attention
            L = sum(self.lens)
            k_start = torch.from_numpy(np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)).cuda()
            every = self.paged.kv_batch(self.n, L, max(self.lens), k_start.data_ptr(), d_len.data_ptr(), self.table.data_ptr())
            kk, vv = (torch.empty(L, KV, D, dtype=TYPES[t_out], device="cuda") for _ in range(2))
            e.kv_gather_dev(self.cfg, every, self.pages.data_ptr(), kk.data_ptr(), vv.data_ptr(), t_out, stream())
            p = self.paged.prompt(H, KV, D, t_out, self.n, T, L, max(news), d_start.data_ptr(), k_start.data_ptr())
            e.attn_prompt_dev(p, qr.data_ptr(), H * D, kk.data_ptr(), KV * D, vv.data_ptr(), KV * D, D ** -0.5, out.data_ptr(),
                              stream())
        torch.cuda.synchronize()
        e.check_device_error()
        # the same, plainly
        pos = np.concatenate([np.arange(l - n, l) for l, n in zip(self.lens, news)]).astype(int)
        qf, kf, vf = (t.cpu().numpy().reshape(T, -1, D) for t in (q, k, v))
        qw = torch.from_numpy(R.rotate(qf, pos, self.cos, self.sin)).to(TYPES[t_out])
        assert torch.equal(qr.cpu(), qw)
        kq, vq = R.values(*R.quantise(R.rotate(kf, pos, self.cos, self.sin))), R.values(*R.quantise(vf))
        for s in range(self.n):
            for i, x64 in enumerate((kq, vq)):
                self.hist[s][i] = np.concatenate([self.hist[s][i], x64[starts[s]:starts[s + 1]]])
        ks, vs = [h[0] for h in self.hist], [h[1] for h in self.hist]
        if prompt_type is None:
            top = max(float(np.abs(x).max(initial=0.0)) for x in vs)
            # (the largest value is 8 times its scale: 2^-28 of the largest scale)
            want, bound = R.attend(qw.double(), ks, vs, news, D ** -0.5, torch.float32, E_SCORE, e_prob(F32), 2.0 ** -31 * top)
        else:
            assert torch.equal(kk.cpu(), torch.from_numpy(np.concatenate(ks)).float().to(TYPES[t_out]))
            assert torch.equal(vv.cpu(), torch.from_numpy(np.concatenate(vs)).float().to(TYPES[t_out]))
            ks, vs = ([torch.from_numpy(x).float().to(TYPES[t_out]).double().numpy() for x in y] for y in (ks, vs))
            want, bound = R.attend(qw.double(), ks, vs, news, D ** -0.5, TYPES[t_out], 2.0 ** -19, e_prob_prompt(t_out),
                                   tiny_prompt(t_out, vv))
        R.check_close(out, want, bound)


@pytest.mark.parametrize("H,KV,D,page,prompt_type", [(8, 2, 64, 16, F16), (6, 6, 128, 48, BF16), (16, 2, 128, 64, F16)])
def test_prompts_then_tokens_then_drafts(engine, pkg, H, KV, D, page, prompt_type):
    """Three prompts at once, one of them empty so far; single tokens while the
    empty one begins; a second prompt behind a cached one; a drafted run."""
    E = 256
    layer = Layer(engine, H, KV, D, E, page, 3, 400, seed=H + D)
    try:
        for i, (news, prompt) in enumerate([([70, 0, 131], True), ([1, 0, 1], False), ([1, 17, 1], False), ([1, 1, 1], False),
                                            ([40, 3, 90], True), ([4, 4, 4], False), ([1, 0, 0], False)]):
            x = rand((sum(news), E), 50 + i).cuda()
            layer.step(news, x, prompt_type if prompt else None)
    finally:
        layer.close()


def test_more_sequences_than_shared_memory_keeps(engine, pkg):
    """1500 sequences, some without new tokens: append, read-back and attention."""
    rng = np.random.default_rng(5)
    news = [int(x) for x in rng.integers(0, 4, 1500)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 30, 1500))]
    pool = Pool(4, 1, 64, 16, lens, news, seed=6, extra_rows=1)
    ks, vs = pool.fill()
    pool.upload()
    q = rand((pool.rows, 4, 64), 7)
    check_paged(engine, pool, ks, vs, q, F32, F32, 0.125)
    check_paged(engine, pool, ks, vs, q.half(), F16, F16, 0.125)
    out = [torch.full((pool.rows, 1, 64), 7.0, device="cuda") for _ in range(2)]
    engine.kv_gather_dev(pool.cfg, pool.batch(), pool.dev["pages"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), F32, stream())
    torch.cuda.synchronize()
    for o, x in zip(out, (ks, vs)):
        want = np.concatenate([r[l - n:] for r, l, n in zip(x, lens, news)])
        assert torch.equal(o[:pool.T].cpu(), torch.from_numpy(want).float()) and (o[pool.T:] == 7.0).all()
    k, v = rand((pool.rows, 1, 64), 8), rand((pool.rows, 1, 64), 9)
    _, cos, sin = run_append(engine, pool, q, k, v, F32, F32, 64)
    kf = R.rotate(k[:pool.T].numpy(), pool.pos(), cos, sin)
    assert np.array_equal(pool.dev["pages"].cpu().numpy(), expected_pages(pool, kf, v[:pool.T].numpy()))
    engine.check_device_error()


@pytest.mark.parametrize("dim,type_", [(64, F16), (128, BF16)])
def test_more_prompts_than_shared_memory_keeps(engine, pkg, dim, type_):
    rng = np.random.default_rng(dim)
    news = [int(x) for x in rng.integers(0, 12, 400)]
    lens = [n + int(x) for n, x in zip(news, rng.integers(0, 40, 400))]
    check_prompt(engine, 4, 2, dim, type_, news, lens, extra=2)


@pytest.mark.parametrize("heads,kv,dim", [(130, 1, 64), (65, 1, 128), (400, 2, 64), (1024, 1024, 64)])
def test_many_heads(engine, pkg, heads, kv, dim):
    """More heads of a K/V head than a tile of rows takes, and the most K/V heads."""
    news, lens = ([5, 40], [5, 200]) if kv < 1024 else ([2, 1], [20, 5])
    check_prompt(engine, heads, kv, dim, BF16, news, lens)
    pool = Pool(heads, kv, dim, 16, lens, [min(n, 3) for n in news])
    ks, vs = pool.fill()
    pool.upload()
    for t in (F32, F16):
        check_paged(engine, pool, ks, vs, rand((pool.rows, heads, dim), 3, t), t, t, dim ** -0.5)


def test_tables_for_lengths_far_beyond_the_cached_ones(engine, pkg):
    """2^30 positions a sequence: the plan's arithmetic is done in coarser units."""
    pool = Pool(8, 4, 64, 4096, [5000, 1, 4096, 300, 17, 9, 4097, 2], [1] * 8, max_pages=1 << 18, spare=0)
    ks, vs = pool.fill()
    pool.upload()
    check_paged(engine, pool, ks, vs, rand((8, 8, 64), 3), F32, F32, 0.125)


def far_pool(pool, n):
    """The pool's pages moved to the end of one of n pages (the rest is not written)."""
    from hf_llm_b200 import paged
    small, m = pool.dev["pages"], pool.n_pages
    big = torch.empty((n,) + tuple(small.shape[1:]), dtype=torch.uint8, device="cuda")
    big[n - m:] = small
    pool.dev["pages"] = big
    pool.dev["table"] += n - m
    pool.cfg = paged.kv_config(pool.H, pool.KV, pool.D, R.Q4_0, pool.P, n, pool.max_pages)
    return n - m


def test_pool_of_more_than_32_bits_of_bytes(engine, pkg):
    H, KV, D = 16, 8, 128
    lens, news = [300, 4100, 33], [3, 1, 33]
    pool = Pool(H, KV, D, 4096, lens, news, spare=0)
    ks, vs = pool.fill()
    pool.upload()
    base = far_pool(pool, (9 << 30) // (KV * 256 * 18 * D))
    assert base * KV * 256 * 18 * D > 2 ** 33
    check_paged(engine, pool, ks, vs, rand((pool.rows, H, D), 3), F32, F32, 0.09)
    out = [torch.empty(pool.rows, KV, D, device="cuda") for _ in range(2)]
    engine.kv_gather_dev(pool.cfg, pool.batch(), pool.dev["pages"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), F32, stream())
    torch.cuda.synchronize()
    for o, x in zip(out, (ks, vs)):
        assert torch.equal(o.cpu(), torch.from_numpy(np.concatenate([r[l - n:] for r, l, n in zip(x, lens, news)])).float())
    k, v = rand((pool.rows, KV, D), 8), rand((pool.rows, KV, D), 9)
    run_append(engine, pool, rand((pool.rows, H, D), 1), k, v, F32, F32, 0)
    assert np.array_equal(pool.dev["pages"][base:].cpu().numpy(), expected_pages(pool, k.numpy(), v.numpy()))
    engine.check_device_error()


def test_rows_further_apart_than_32_bits_of_elements(engine, pkg):
    """Rows of 2^31 elements: the third starts 2^32 elements behind the first."""
    from hf_llm_b200 import paged
    H, KV, D, n, far = 4, 2, 64, 3, 1 << 31
    pool = Pool(H, KV, D, 16, [n], [n], spare=0).upload()
    big = torch.empty(2 * far + 512, dtype=torch.float16, device="cuda")
    at = [0, 256, 384]
    x = [rand((n, h, D), 3 + i, F16) for i, h in enumerate((H, KV, KV))]
    for a, y in zip(at, x):
        for i in range(n):
            big[i * far + a:i * far + a + y[i].numel()] = y[i].reshape(-1).cuda()
    ptr = [big.data_ptr() + 2 * a for a in at]
    q_out = torch.empty(n, H, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    engine.kv_append_dev(pool.cfg, pool.batch(), None, F16, ptr[0], far, ptr[1], far, ptr[2], far, pool.dev["pages"].data_ptr(),
                         q_out.data_ptr(), F16, stream())
    torch.cuda.synchronize()
    assert torch.equal(q_out.cpu(), x[0])
    assert np.array_equal(pool.dev["pages"].cpu().numpy(), expected_pages(pool, x[1].float().numpy(), x[2].float().numpy()))
    got = run_paged(engine, pool, x[0], F16, F16, 0.125)
    b = pool.batch()
    work = torch.empty(engine.attn_paged_work_bytes(pool.cfg, b), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(got)
    engine.attn_paged_dev(pool.cfg, b, ptr[0], F16, far, pool.dev["pages"].data_ptr(), 0.125, out.data_ptr(), F16,
                          work.data_ptr(), work.numel(), stream())
    torch.cuda.synchronize()
    assert torch.equal(out, got)
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    p = paged.prompt(H, KV, D, F16, 1, n, n, n, start.data_ptr(), start.data_ptr())
    outs = []
    for ptrs, st in ((ptr, (far,) * 3), ([y.cuda() for y in x], (H * D, KV * D, KV * D))):
        keep = ptrs
        o = torch.full((n, H, D), 7.0, dtype=torch.float16, device="cuda")
        ad = [y if isinstance(y, int) else y.data_ptr() for y in keep]
        torch.cuda.synchronize()
        engine.attn_prompt_dev(p, ad[0], st[0], ad[1], st[1], ad[2], st[2], 0.125, o.data_ptr(), stream())
        torch.cuda.synchronize()
        outs.append(o)
    assert torch.equal(*outs)
    engine.check_device_error()


def test_offsets_that_count_the_rows_again_and_again(engine, pkg):
    """300 of 600 sequences claim all rows with 2^22 keys each: above 2^31 units of
    work, which is reported and not begun."""
    from hf_llm_b200 import paged
    from hf_llm_b200._lib import B2QError, EINVAL
    H, D, T, S, P, mp = 4, 64, 64, 600, 4096, 1024
    cfg = paged.kv_config(H, H, D, R.Q4_0, P, 1, mp)
    start = torch.tensor([0, T] * (S // 2) + [0], dtype=torch.int32).cuda()
    lens = torch.full((S,), mp * P, dtype=torch.int32).cuda()
    table = torch.full((S, mp), -1, dtype=torch.int32).cuda()
    pages = torch.empty(paged.page_bytes(cfg), dtype=torch.uint8, device="cuda")
    b = paged.kv_batch(S, T, 1, start.data_ptr(), lens.data_ptr(), table.data_ptr())
    assert 300 * (T // 8) * H * (mp * P // 16 + 5) > 2 ** 31
    q = rand((T, H, D), 1).cuda()
    out = torch.full_like(q, 7.0)
    work = torch.empty(engine.attn_paged_work_bytes(cfg, b), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    engine.attn_paged_dev(cfg, b, q.data_ptr(), F32, H * D, pages.data_ptr(), 0.125, out.data_ptr(), F32, work.data_ptr(),
                          work.numel(), stream())
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    with pytest.raises(B2QError) as e:
        engine.check_device_error()
    assert e.value.status == EINVAL


def test_two_prompt_calls_at_once(engine, pkg):
    """The same packed prompts on two streams at the same time, several calls each."""
    from hf_llm_b200 import paged
    H, KV, D, news = 8, 2, 128, [300, 17, 129]
    T = sum(news)
    start = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32).cuda()
    p = paged.prompt(H, KV, D, BF16, 3, T, T, 300, start.data_ptr(), start.data_ptr())
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
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    engine.check_device_error()
