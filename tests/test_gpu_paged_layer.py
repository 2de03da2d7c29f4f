"""One attention layer as the integration notes write it down: projections, append, read-back,
packed prompt attention, widening and the output product; and the same for single tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R
from paged_ref import BF16, F16, F32, TYPES
from test_gpu_paged import rand

pytestmark = pytest.mark.gpu

Q8_0 = 8


def weight(engine, rng, n, k):
    code = rng.integers(-127, 128, (n, k // 32, 32)).astype(np.int8)
    scale = np.full((n, k // 32, 1), 1 / (73 * np.sqrt(k)), np.float16)
    raw = np.concatenate([scale.view(np.uint8).reshape(n, k // 32, 2), code.view(np.uint8)], -1)
    return (code * scale.astype(np.float64)).reshape(n, k), engine.try_upload_weight(raw.reshape(-1), Q8_0, n, k)


@pytest.mark.parametrize("type_", [F16, BF16])
def test_the_documented_step(engine, pkg, type_):
    from hf_llm_b200 import paged
    H, KV, D, E, P = 8, 2, 64, 256, 16
    rng = np.random.default_rng(3)
    (wq, bq), (wk, bk), (wv, bv), (wo, bo) = (weight(engine, rng, n, k) for n, k in ((H * D, E), (KV * D, E), (KV * D, E), (E, H * D)))
    S, room = 3, 256
    mp = room // P
    cfg = paged.kv_config(H, KV, D, R.Q4_0, P, S * mp, mp)
    table = torch.from_numpy(rng.permutation(S * mp).astype(np.int32).reshape(S, mp)).cuda()
    pages = torch.full((S * mp * paged.page_bytes(cfg),), 0xff, dtype=torch.uint8, device="cuda")
    cos, sin = R.rope_tables(room, D)
    tables = [torch.from_numpy(x).cuda() for x in (cos, sin)]
    rope = paged.rope(D, room, *(x.data_ptr() for x in tables))
    lens, hist = [0] * S, [[np.zeros((0, KV, D))] * 2 for _ in range(S)]
    st = 1
    try:
        for news, prompt in (([40, 3, 100], True), ([1, 1, 1], False), ([30, 0, 64], True)):
            T = sum(news)
            lens = [a + b for a, b in zip(lens, news)]
            x = rand((T, E), 7 + T).cuda()
            y = torch.empty(T * (H + 2 * KV) * D, device="cuda")
            start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
            q_start, kv_len = torch.from_numpy(start).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
            t = type_ if prompt else F32
            q_out = torch.empty(T, H, D, dtype=TYPES[t], device="cuda")
            out, wide, z = torch.empty_like(q_out), torch.empty(T, H * D, device="cuda"), torch.empty(T, E, device="cuda")
            batch = paged.kv_batch(S, T, max(news), q_start.data_ptr(), kv_len.data_ptr(), table.data_ptr())
            torch.cuda.synchronize()
            engine.matmul_group_dev([(bq, H * D), (bk, KV * D), (bv, KV * D)], x.data_ptr(), y.data_ptr(), T, E, st)
            q, k, v = (y[a * T:b * T].view(T, b - a) for a, b in ((0, H * D), (H * D, (H + KV) * D), ((H + KV) * D, (H + 2 * KV) * D)))
            engine.kv_append_dev(cfg, batch, rope, F32, q.data_ptr(), H * D, k.data_ptr(), KV * D, v.data_ptr(), KV * D, pages.data_ptr(),
                                 q_out.data_ptr(), t, st)
            if prompt:
                L = sum(lens)
                sums = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
                every = paged.kv_batch(S, L, max(lens), sums.data_ptr(), kv_len.data_ptr(), table.data_ptr())
                k16, v16 = (torch.empty(L, KV, D, dtype=TYPES[t], device="cuda") for _ in range(2))
                torch.cuda.synchronize()
                engine.kv_gather_dev(cfg, every, pages.data_ptr(), k16.data_ptr(), v16.data_ptr(), t, st)
                p = paged.prompt(H, KV, D, t, S, T, L, max(news), q_start.data_ptr(), sums.data_ptr())
                engine.attn_prompt_dev(p, q_out.data_ptr(), H * D, k16.data_ptr(), KV * D, v16.data_ptr(), KV * D, D ** -0.5, out.data_ptr(), st)
                engine.dequantize_dev(out.data_ptr(), t, out.numel(), wide.data_ptr(), st)
            else:
                work = torch.empty(engine.attn_paged_work_bytes(cfg, batch), dtype=torch.uint8, device="cuda")
                engine.attn_paged_dev(cfg, batch, q_out.data_ptr(), F32, H * D, pages.data_ptr(), D ** -0.5, wide.data_ptr(), F32,
                                      work.data_ptr(), work.numel(), st)
            engine.matmul_dev(bo, wide.data_ptr(), z.data_ptr(), T, E, H * D, st)
            torch.cuda.synchronize()
            engine.check_device_error()
            # the layer in f64, from the projections as the products gave them (codes hang on their roundings)
            pos = np.concatenate([np.arange(l - n, l) for l, n in zip(lens, news)]).astype(int)
            qf, kf, vf = (r.cpu().numpy().reshape(T, -1, D) for r in (q, k, v))
            kq, vq = R.values(*R.quantise(R.rotate(kf, pos, cos, sin))), R.values(*R.quantise(vf))
            for s in range(S):
                hist[s] = [np.concatenate([h, r[start[s]:start[s + 1]]]) for h, r in zip(hist[s], (kq, vq))]
            qr = torch.from_numpy(R.rotate(qf, pos, cos, sin)).double()
            o, _ = R.attend(qr, [h[0] for h in hist], [h[1] for h in hist], news, D ** -0.5, TYPES[t], 0.0, 0.0)
            for got, w in ((q, wq), (k, wk), (v, wv)):  # (products: relative to their norm, as their own tests)
                want = x.cpu().double().numpy() @ w.T
                assert np.linalg.norm(got.cpu().numpy() - want) <= 1e-3 * np.linalg.norm(want)
            # 16-bit queries and keys move a score by 2 half steps of sum |q k| / 8 (about 5 for rows of unit size) and a
            # weight by twice that, 20 half steps; values, probabilities and outputs are rounded once each; 1e-3 of the product
            tol = 1e-3 + (24 * R.half_eps(TYPES[t]) if prompt else 1e-5)
            want = o.numpy().reshape(T, H * D) @ wo.T
            assert np.linalg.norm(z.cpu().numpy() - want) <= tol * np.linalg.norm(want)
    finally:
        for b in (bq, bk, bv, bo):
            b.free()
