"""The paged 4-bit K/V cache operators on a B200 (b2q_kv_append_dev,
b2q_kv_gather_dev, b2q_attn_paged_dev) against plain statements of them: what
the append writes byte by byte and the read-back bit by bit, attention within
bounds derived from its roundings (paged_ref.attend)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, F32, Pool, TYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=[0, 4000], ids=["short table", "long table"])
def table(request):
    """What a page table has room for decides how few sequences are divided among
    the CTAs: an item to a cluster, or all of them as one line."""
    R.MORE_PAGES = request.param
    yield
    R.MORE_PAGES = 0



def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def rand(shape, seed, type_=F32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(TYPES[type_])


def run_append(engine, pool, q, k, v, x_type, out_type, rot, n_pos=None, strided=False):
    from hf_llm_b200 import paged
    n_pos = n_pos or max(1, max(pool.lens))
    cos, sin = R.rope_tables(n_pos, rot or 8)
    cd, sd = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
    H, KV, D = pool.H, pool.KV, pool.D
    if strided:  # one row of q | k | v for every token
        row = torch.cat([q.reshape(len(q), -1), k.reshape(len(k), -1), v.reshape(len(v), -1)], 1).cuda().contiguous()
        st = (row.shape[1],) * 3
        es = row.element_size()
        ptrs = (row.data_ptr(), row.data_ptr() + H * D * es, row.data_ptr() + (H + KV) * D * es)
    else:
        keep = [x.cuda().contiguous() for x in (q, k, v)]
        st = (H * D, KV * D, KV * D)
        ptrs = tuple(x.data_ptr() for x in keep)
    q_out = torch.full((pool.rows, H, D), 7.0, dtype=TYPES[out_type], device="cuda")
    torch.cuda.synchronize()
    engine.kv_append_dev(pool.cfg, pool.batch(), paged.rope(rot, n_pos, cd.data_ptr(), sd.data_ptr()) if rot else None, x_type,
                         ptrs[0], st[0], ptrs[1], st[1], ptrs[2], st[2], pool.dev["pages"].data_ptr(), q_out.data_ptr(), out_type,
                         stream())
    torch.cuda.synchronize()
    return q_out, cos, sin


def expected_pages(pool, k, v):
    """The pool's bytes after the append of f32 rows k, v [T, KV, D]."""
    pages = pool.pages.copy()
    D = pool.D
    (kc, ks), (vc, vs) = R.quantise(k), R.quantise(v)
    mask = np.ones((16, D), np.uint8) * 15
    ff = np.full((16, D // 32), 0xffff, np.uint16).view(np.float16)
    zc, zs = np.zeros((16, D), np.uint8), np.zeros((16, D // 32), np.float16)
    for t, (s, p) in enumerate(zip(pool.seq(), pool.pos())):
        for h in range(pool.KV):
            blk = pages[pool.table[s, p // pool.P], h, p % pool.P // 16]
            part = []
            own = []
            for c, d in ((kc, ks), (vc, vs)):
                ci, di, mi, fi = zc.copy(), zs.copy(), zc.copy(), zs.copy()
                ci[p % 16], di[p % 16] = c[t, h], d[t, h]
                mi[p % 16], fi[p % 16] = mask[0], ff[0]
                part += [ci, di]
                own += [mi, fi]
            new, mine = R.block_bytes(*part), R.block_bytes(*own)
            blk[:] = (blk & ~mine) | (new & mine)
    return pages


def nan_scales_equal(a, b, D):
    """Bytes equal, but any NaN scale equals any other."""
    same = a == b
    for o in (8 * D, 17 * D):
        x = np.isnan(np.ascontiguousarray(a[..., o:o + D]).view(np.float16))
        y = np.isnan(np.ascontiguousarray(b[..., o:o + D]).view(np.float16))
        same[..., o:o + D] |= np.repeat(x & y, 2, -1)
    return same.all()


@pytest.mark.parametrize("heads,kv,dim,page,lens,news,x_type,out_type,rot,strided", [
    (8, 2, 128, 16, [1], [1], F32, F32, 128, False),
    (8, 2, 128, 64, [5, 130, 0, 77], [1, 7, 0, 77], F32, F16, 128, True),
    (4, 4, 64, 32, [33, 64, 65], [2, 64, 1], F16, BF16, 64, True),
    (6, 2, 64, 48, [100, 47], [50, 3], BF16, BF16, 32, False),
    (5, 5, 64, 16, [17, 9], [17, 9], F32, F16, 24, False),   # odd head count, partial rotation
    (12, 4, 128, 256, [300, 1, 256], [19, 1, 0], F16, F16, 0, False),
    (32, 8, 128, 64, [700] * 3, [1] * 3, BF16, F32, 128, False),
])
def test_append_writes_the_documented_bytes(engine, pkg, heads, kv, dim, page, lens, news, x_type, out_type, rot, strided):
    pool = Pool(heads, kv, dim, page, lens, news, seed=5, extra_rows=3).upload()
    q, k, v = (rand((pool.rows, h, dim), 10 + i, x_type) for i, h in enumerate((heads, kv, kv)))
    k[0, 0, :32] = 0.0  # a block of zeros
    v[0, 0, :2] = torch.tensor([3.0, -3.0]) * 2  # the largest magnitude twice, signs apart
    q_out, cos, sin = run_append(engine, pool, q, k, v, x_type, out_type, rot, strided=strided)
    qf, kf, vf = (x[:pool.T].float().numpy() for x in (q, k, v))
    if rot:
        qf, kf = R.rotate(qf, pool.pos(), cos, sin), R.rotate(kf, pool.pos(), cos, sin)
    assert torch.equal(q_out[:pool.T].cpu(), torch.from_numpy(qf).to(TYPES[out_type]))
    assert (q_out[pool.T:] == 7.0).all()  # rows behind the last sequence
    assert np.array_equal(pool.dev["pages"].cpu().numpy(), expected_pages(pool, kf, vf))
    engine.check_device_error()


def test_append_extreme_values(engine, pkg):
    """Infinities and NaN poison their block of 32 only; huge magnitudes keep a
    finite scale; magnitudes below the smallest scale give zeros."""
    pool = Pool(2, 2, 128, 16, [3], [3], extra_rows=0).upload()
    k, v, q = (rand((3, 2, 128), s) for s in (1, 2, 3))
    k[0, 0, 40] = float("inf")
    k[1, 1, 0] = float("nan")
    v[0, 1, 127] = -float("inf")
    v[1, 0] *= 1e6
    v[2, 0] *= 1e-9
    v[2, 1] *= 3e-7
    v[0, 0] *= 1e38
    run_append(engine, pool, q, k, v, F32, F32, 0)
    got = pool.dev["pages"].cpu().numpy()
    assert nan_scales_equal(got, expected_pages(pool, k.numpy(), v.numpy()), 128)


def test_append_without_queries_and_in_place(engine, pkg):
    from hf_llm_b200 import paged
    pool = Pool(4, 2, 64, 16, [40], [40]).upload()
    q, k, v = (rand((40, h, 64), 3 + i, F16) for i, h in enumerate((4, 2, 2)))
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    cos, sin = (torch.from_numpy(x).cuda() for x in R.rope_tables(64, 64))
    rope = paged.rope(64, 64, cos.data_ptr(), sin.data_ptr())
    p = pool.dev["pages"].data_ptr()
    engine.kv_append_dev(pool.cfg, pool.batch(), rope, F16, 0, 0, kd.data_ptr(), 128, vd.data_ptr(), 128, p, 0, F16, stream())
    first = pool.dev["pages"].clone()
    engine.kv_append_dev(pool.cfg, pool.batch(), rope, F16, qd.data_ptr(), 256, kd.data_ptr(), 128, vd.data_ptr(), 128, p,
                         qd.data_ptr(), F16, stream())
    torch.cuda.synchronize()
    assert torch.equal(first, pool.dev["pages"])
    want = R.rotate(q.float().numpy(), pool.pos(), cos.cpu().numpy(), sin.cpu().numpy())
    assert torch.equal(qd.cpu(), torch.from_numpy(want).half())


@pytest.mark.parametrize("kv,dim,page,lens,news,out_type", [
    (2, 128, 64, [100, 1, 0, 64], [100, 1, 0, 64], F32),
    (3, 64, 16, [33, 250], [5, 249], F16),
    (8, 128, 48, [47, 49, 500], [47, 0, 333], BF16),
    (1, 64, 256, [1], [1], F32),
])
def test_gather_reads_back_what_is_cached(engine, pkg, kv, dim, page, lens, news, out_type):
    pool = Pool(kv, kv, dim, page, lens, news, extra_rows=2)
    ks, vs = pool.fill()
    pool.upload()
    out = [torch.full((pool.rows, kv, dim), 7.0, dtype=TYPES[out_type], device="cuda") for _ in range(2)]
    engine.kv_gather_dev(pool.cfg, pool.batch(), pool.dev["pages"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out_type,
                         stream())
    torch.cuda.synchronize()
    for o, x in zip(out, (ks, vs)):
        want = torch.from_numpy(np.concatenate([r[l - n:] for r, l, n in zip(x, lens, news)])).float().to(TYPES[out_type])
        assert torch.equal(o[:pool.T].cpu(), want)
        assert (o[pool.T:] == 7.0).all()
    one = torch.empty(pool.rows, kv, dim, dtype=TYPES[out_type], device="cuda")
    engine.kv_gather_dev(pool.cfg, pool.batch(), pool.dev["pages"].data_ptr(), 0, one.data_ptr(), out_type, stream())
    torch.cuda.synchronize()
    assert torch.equal(one[:pool.T], out[1][:pool.T])
    engine.check_device_error()


def run_paged(engine, pool, q, q_type, out_type, scale, max_new=None, work=None, q_stride=None):
    q = q.cuda()
    out = torch.full((pool.rows, pool.H, pool.D), 7.0, dtype=TYPES[out_type], device="cuda")
    b = pool.batch(max_new)
    if work is None:
        work = torch.full((engine.attn_paged_work_bytes(pool.cfg, b),), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    engine.attn_paged_dev(pool.cfg, b, q.data_ptr(), q_type, q_stride or pool.H * pool.D, pool.dev["pages"].data_ptr(), scale,
                          out.data_ptr(), out_type, work.data_ptr(), work.numel(), stream())
    torch.cuda.synchronize()
    return out


# f32 queries as two f16 parts: 2^-21 of each product, and f32 sums of them over
# the head; 16-bit queries enter exactly.  A probability times its scale is two
# f16 parts where the output is f32 (2^-21), and one, rounded once (2^-11, as
# f16 half a step), for 16-bit outputs
E_SCORE = 2.0 ** -20


def e_prob(out_type):
    return 2.0 ** -21 if out_type == F32 else 2.0 ** -11


def tiny(pool):
    """A probability times its scale, 2^6 or above for a probability of 1 and the
    largest scale, is off by at most half of f16's smallest step, 2^-25, as well,
    so a term by 2^-31 of the largest scale times |code - 8| <= 8; the sum of the
    probabilities is at least 1."""
    return 2.0 ** -28 * pool.largest_scale()




def check_paged(engine, pool, ks, vs, q, q_type, out_type, scale, **kw):
    out = run_paged(engine, pool, q, q_type, out_type, scale, **kw)
    want, bound = R.attend(q[:pool.T].double(), ks, vs, pool.news, scale, TYPES[out_type], E_SCORE, e_prob(out_type), tiny(pool))
    R.check_close(out[:pool.T], want, bound)
    assert (out[pool.T:] == 7.0).all()
    engine.check_device_error()
    return out


@pytest.mark.parametrize("heads,kv,dim,page,lens,news,q_type,out_type", [
    (8, 2, 128, 16, [1], [1], F32, F32),
    (8, 2, 128, 64, [15, 16, 17, 63, 64, 65], [1] * 6, F32, F32),
    (32, 8, 128, 64, [585], [1], F16, F16),
    (16, 16, 64, 48, [100, 7, 333], [1, 2, 3], BF16, BF16),
    (24, 8, 128, 32, [257, 1, 0, 40], [5, 1, 0, 8], F16, F32),
    (9, 1, 64, 16, [129, 31], [1, 7], F32, F16),
    (64, 8, 128, 256, [700, 3], [5, 3], BF16, F32),
    (32, 1, 128, 16, [95], [2], F32, BF16),
    (40, 8, 64, 64, [130, 500, 20], [33, 1, 20], F32, F32),   # more rows than one tile of queries
    (4, 4, 128, 16, [3000], [1], F32, F32),
    (8, 1, 128, 64, [2500, 10, 1, 900], [1, 1, 1, 1], F16, F16),
    (2, 2, 64, 32, [5] * 150, [1] * 150, F32, F32),            # many short sequences
])
def test_attention_over_the_cache(engine, pkg, heads, kv, dim, page, lens, news, q_type, out_type):
    pool = Pool(heads, kv, dim, page, lens, news, seed=3, extra_rows=2)
    ks, vs = pool.fill()
    pool.upload()
    q = rand((pool.rows, heads, dim), 9, q_type)
    scale = dim ** -0.5
    out = check_paged(engine, pool, ks, vs, q, q_type, out_type, scale)
    for hint in (0, 1, 64):  # the hint never changes what a row attends
        check_paged(engine, pool, ks, vs, q, q_type, out_type, scale, max_new=hint)
    assert torch.equal(out, run_paged(engine, pool, q, q_type, out_type, scale))  # the same bits every time


@pytest.mark.parametrize("q_spread,v_spread,scale", [(30.0, 1.0, 0.09), (1e-4, 1.0, 0.09), (3e4, 1e-3, 1e-5), (1.0, 1e-5, 0.3), (1.0, 200.0, 0.01)])
def test_attention_far_from_unit_size(engine, pkg, q_spread, v_spread, scale):
    """Peaked and flat softmaxes, values near f16's smallest and large scales."""
    pool = Pool(8, 2, 128, 64, [200, 65], [1, 4])
    ks, vs = pool.fill(spread=v_spread)
    pool.upload()
    q = rand((pool.rows, 8, 128), 2, F32, q_spread / v_spread ** 0.5)
    check_paged(engine, pool, ks, vs, q, F32, F32, scale)


def test_attention_scales_of_very_different_size(engine, pkg):
    """Values whose scales differ by 2^20 between tokens and blocks of dims."""
    pool = Pool(4, 1, 128, 16, [333], [3])
    ks, vs = pool.fill()
    rng = np.random.default_rng(0)
    blk = pool.pages.reshape(-1, 18 * 128)
    f = (2.0 ** rng.integers(-12, 9, (len(blk), 64))).astype(np.float32)
    vsc = blk[:, 17 * 128:].copy().view(np.float16)
    new = (vsc.astype(np.float32) * f).astype(np.float16)
    new[~np.isfinite(vsc.astype(np.float32))] = np.nan
    blk[:, 17 * 128:] = new.view(np.uint8)
    pool.pages = blk.reshape(pool.pages.shape)
    # the values again, read from the bytes
    v = np.zeros((333, 1, 128))
    for p in range(333):
        b = pool.pages[pool.table[0, p // 16], 0, 0]
        for d in range(128):
            byte = b[9 * 128 + p % 16 // 8 * 512 + d % 8 * 64 + p % 8 // 2 * 16 + p % 2 * 8 + d // 16]
            code = int(byte >> (4 * (d // 8 % 2))) & 15
            v[p, 0, d] = (code - 8) * float(b[17 * 128:].view(np.float16)[p % 16 * 4 + d // 32])
    pool.upload()
    check_paged(engine, pool, ks, [v], rand((3, 4, 128), 4), F32, F32, 0.09)


def test_a_poisoned_sequence_stays_alone(engine, pkg):
    """NaN blocks of one sequence do not reach another's rows, nor the rows of
    the same sequence whose position lies before them."""
    pool = Pool(4, 2, 64, 16, [50, 50], [4, 4])
    ks, vs = pool.fill()
    clean = pool.pages.copy()
    last = pool.pages[pool.table[0, 48 // 16], :, 0]
    for o in (8 * 64, 17 * 64):  # the scales of position 48 of sequence 0
        last[:, o:o + 64].reshape(2, 16, 4)[:, 0] = 0xff
    pool.upload()
    q = rand((8, 4, 64), 5)
    out = run_paged(engine, pool, q, F32, F32, 0.125)
    assert torch.isfinite(out[:2]).all() and torch.isnan(out[2:4]).all() and torch.isfinite(out[4:]).all()
    pool.pages = clean
    pool.upload()
    ok = run_paged(engine, pool, q, F32, F32, 0.125)
    assert torch.equal(out[:2], ok[:2]) and torch.equal(out[4:], ok[4:])


def test_shared_pages_and_one_query_set_twice(engine, pkg):
    """Two sequences with the same pages (a shared beginning) and the same
    queries; where the work is cut differs between them, so the sums' order may."""
    pool = Pool(8, 2, 128, 16, [100, 100], [2, 2])
    ks, vs = pool.fill()
    pool.table[1] = pool.table[0]
    pool.upload()
    q = rand((2, 8, 128), 5)
    q = torch.cat([q, q])
    check_paged(engine, pool, [ks[0]] * 2, [vs[0]] * 2, q, F32, F32, 0.09)


def test_strided_queries(engine, pkg):
    pool = Pool(8, 2, 64, 16, [70, 3], [1, 1])
    ks, vs = pool.fill()
    pool.upload()
    wide = rand((2, 8 * 64 + 256), 5, F16)
    q = wide[:, :512].reshape(2, 8, 64)
    out = run_paged(engine, pool, wide, F16, F32, 0.125, q_stride=768)
    want, bound = R.attend(q.double(), ks, vs, pool.news, 0.125, torch.float32, E_SCORE, e_prob(F32), tiny(pool))
    R.check_close(out, want, bound)


def test_bad_positions_pages_and_offsets_are_skipped_and_reported(engine, pkg):
    from hf_llm_b200._lib import B2QError, EINVAL

    def expect_error():
        with pytest.raises(B2QError) as e:
            engine.check_device_error()
        assert e.value.status == EINVAL
        engine.check_device_error()  # once

    pool = Pool(4, 2, 64, 16, [40, 40], [2, 2])
    ks, vs = pool.fill()
    clean = pool.pages.copy()
    q, k, v = rand((4, 4, 64), 1), rand((4, 2, 64), 2), rand((4, 2, 64), 3)
    good = run_paged(engine, pool.upload(), q, F32, F32, 0.125)
    want, bound = R.attend(q[2:].double(), ks[1:], vs[1:], [2], 0.125, torch.float32, E_SCORE, e_prob(F32), tiny(pool))
    for bad in (-1, pool.n_pages, 2 ** 31 - 1, -2 ** 31):
        for page in (0, 2):
            pool.table[0, page] = bad
            pool.upload()
            out = run_paged(engine, pool, q, F32, F32, 0.125)
            assert torch.isfinite(out).all() and torch.equal(out[2:], good[2:])
            expect_error()
            run_append(engine, pool, q, k, v, F32, F32, 64)
            if page == 2:  # the new tokens' page
                expect_error()
            pool.table[0] = Pool(4, 2, 64, 16, [40, 40], [2, 2]).table[0]
            pool.pages = clean.copy()
    for lens in ([1, 40], [-5, 40], [10 ** 9, 40], [-2 ** 31, 40]):  # fewer cached tokens than new ones; more than pages
        p2 = Pool(4, 2, 64, 16, [40, 40], [2, 2])
        p2.fill()
        p2.lens = lens
        p2.upload()
        before = p2.dev["pages"].clone()
        out = run_paged(engine, p2, q, F32, F32, 0.125)
        R.check_close(out[2:], want, bound)  # (not the same bits: the other's length moves the cuts of the work)
        expect_error()
        run_append(engine, p2, q, k, v, F32, F32, 64, n_pos=64)
        expect_error()
        # sequence 1's rows are written, and nothing outside the pages of either
        mine = torch.zeros(p2.n_pages, dtype=torch.bool, device="cuda")
        mine[torch.from_numpy(p2.table[:, :3].reshape(-1).astype(np.int64)).cuda()] = True
        assert torch.equal(p2.dev["pages"][~mine], before[~mine])
    # a decreasing offset leaves a sequence without rows; one out of range is reported
    for starts in ([0, 3, 2], [0, -4, 4], [5, 2, 4], [0, 2 ** 31 - 1, 4], [-2 ** 31, 2, 4]):
        p3 = Pool(4, 2, 64, 16, [40, 40], [2, 2])
        p3.fill()
        p3.q_start = np.array(starts, np.int32)
        p3.upload()
        run_paged(engine, p3, q, F32, F32, 0.125)
        run_append(engine, p3, q, k, v, F32, F32, 64, n_pos=64)
        if starts == [0, 3, 2]:
            try:
                engine.check_device_error()
            except B2QError as e:
                assert e.status == EINVAL
        else:
            expect_error()
    # a rotation table that ends before the position
    p4 = Pool(4, 2, 64, 16, [40], [2]).upload()
    run_append(engine, p4, q, k, v, F32, F32, 64, n_pos=39)
    expect_error()
    keys = p4.dev["pages"][p4.table[0, 2], :, 0, :512].view(2, 16, 32)
    assert (keys[:, 6] != 0xff).any() and (keys[:, 7] == 0xff).all()  # position 38 is written, 39 is not


def test_empty_calls(engine, pkg):
    pool = Pool(4, 2, 64, 16, [40], [0], extra_rows=2)
    pool.fill()
    pool.upload()
    q = rand((2, 4, 64), 1)
    out = run_paged(engine, pool, q, F32, F32, 0.125)
    assert (out == 7.0).all()
    q_out, _, _ = run_append(engine, pool, q, rand((2, 2, 64), 2), rand((2, 2, 64), 3), F32, F32, 64)
    assert (q_out == 7.0).all() and np.array_equal(pool.dev["pages"].cpu().numpy(), pool.pages)
    pool.rows = 0
    run_paged(engine, pool, q, F32, F32, 0.125)
    engine.check_device_error()


def test_two_streams_and_a_replayed_graph(engine, pkg):
    """Calls on two streams at once with a workspace each, and a decode step
    (append, attention) captured once and replayed as the sequences grow: the
    bits of calls made one by one."""
    from hf_llm_b200 import paged
    H, KV, D = 8, 2, 128
    lens, steps = [20, 61, 5], 6
    pools = [Pool(H, KV, D, 16, [l + steps for l in lens], [1] * 3, seed=4) for _ in range(3)]
    for p in pools:
        p.fill(seed=8)
        p.upload()
    cos, sin = (torch.from_numpy(x).cuda() for x in R.rope_tables(128, D))
    rope = paged.rope(D, 128, cos.data_ptr(), sin.data_ptr())
    xs = [[rand((3, h, D), 100 * i + j).cuda() for j, h in enumerate((H, KV, KV))] for i in range(steps)]
    bufs = [[torch.empty_like(x) for x in xs[0]] for _ in pools]
    qo = [torch.empty(3, H, D, device="cuda") for _ in pools]
    out = [torch.empty(3, H, D, device="cuda") for _ in pools]
    work = [torch.full((engine.attn_paged_work_bytes(p.cfg, p.batch()),), 0xff, dtype=torch.uint8, device="cuda") for p in pools]

    def step(i, st):
        p, (q, k, v) = pools[i], bufs[i]
        engine.kv_append_dev(p.cfg, p.batch(), rope, F32, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D,
                             p.dev["pages"].data_ptr(), qo[i].data_ptr(), F32, st)
        engine.attn_paged_dev(p.cfg, p.batch(), qo[i].data_ptr(), F32, H * D, p.dev["pages"].data_ptr(), 0.09, out[i].data_ptr(),
                              F32, work[i].data_ptr(), work[i].numel(), st)

    def set_len(i, n):
        pools[i].dev["kv_len"].copy_(torch.tensor([l + n for l in lens], dtype=torch.int32))

    want = []
    for n in range(steps):
        for b, x in zip(bufs[0], xs[n]):
            b.copy_(x)
        set_len(0, n + 1)
        torch.cuda.synchronize()
        step(0, 1)
        torch.cuda.synchronize()
        want.append(out[0].clone())
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    set_len(1, 1)
    for b, x in zip(bufs[1], xs[0]):
        b.copy_(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s1):
        step(1, s1.cuda_stream)
    for n in range(steps):
        for i in (1, 2):
            set_len(i, n + 1)
            for b, x in zip(bufs[i], xs[n]):
                b.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g.replay()
        step(2, s2.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(out[1], want[n]) and torch.equal(out[2], want[n]), n
    engine.check_device_error()
