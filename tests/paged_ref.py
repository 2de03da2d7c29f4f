"""Plain statements, in numpy and torch on the CPU, of the paged 4-bit K/V
cache, its rotation and quantisation (step by step in f32, as the entry
points document them), and of attention in f64 with an error bound of each
output; and a pool of pages with the device arrays of a batch."""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

TYPES = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
F32, F16, Q4_0, BF16 = 0, 1, 2, 30


def half_eps(t) -> float:
    """Largest relative error of one rounding to torch type t."""
    return torch.finfo(t).eps / 2


def rope_tables(n_pos: int, rot: int, theta: float = 1e4):
    ang = np.arange(n_pos)[:, None] * theta ** (-np.arange(0, rot, 2) / rot)[None, :]
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rotate(x: np.ndarray, pos: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [T, heads, D] f32, each product and sum rounded to f32."""
    r = cos.shape[1]
    y = x.copy()
    a, b = x[..., :r], x[..., r:2 * r]
    c, s = cos[pos][:, None], sin[pos][:, None]
    y[..., :r] = a * c - b * s
    y[..., r:2 * r] = b * c + a * s
    return y


def quantise(x: np.ndarray):
    """Codes [..., D] and f16 scales [..., D / 32] of f32 values."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    finite = np.isfinite(b).all(-1)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
        d = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16)
        df = d.astype(np.float32)
        code = np.clip(np.rint(np.where(df == 0, np.float32(0), b / df)) + 8, 0, 15)
    code = np.where(finite[..., None], code, 8).astype(np.uint8)
    d = d[..., 0]
    d[~finite] = np.nan
    return code.reshape(x.shape), d


def values(code: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """f64 values of codes [..., D] with scales [..., D / 32]."""
    b = code.reshape(*scale.shape, 32).astype(np.float64) - 8
    return (b * scale.astype(np.float64)[..., None]).reshape(code.shape)


@functools.lru_cache(maxsize=None)
def _places(D: int):
    """Where the 4-bit codes [16, D] of keys and values go: indices of half bytes."""
    tok, dim = np.arange(16)[:, None], np.arange(D)[None, :]
    b, t, n = dim // 32, dim % 32 // 8, dim % 8
    keys = 2 * (tok * D // 2 + t * (D // 8) + b * 4 + n // 2) + n % 2
    g, j = dim % 8, dim // 8
    vals = 2 * (9 * D + tok // 8 * 4 * D + g * D // 2 + tok % 8 // 2 * (D // 8) + tok % 2 * (D // 16) + j // 2) + j % 2
    return keys, vals


def block_bytes(kc, ks, vc, vs) -> np.ndarray:
    """One block's bytes: kc, vc [16, D] codes, ks, vs [16, D / 32] f16."""
    D = kc.shape[1]
    half = np.zeros(36 * D, np.uint8)
    keys, vals = _places(D)
    half[keys], half[vals] = kc, vc
    out = half[0::2] | half[1::2] << 4
    out[8 * D:9 * D] = np.ascontiguousarray(ks, np.float16).view(np.uint8).reshape(-1)
    out[17 * D:] = np.ascontiguousarray(vs, np.float16).view(np.uint8).reshape(-1)
    return out


MORE_PAGES = 0  # unused entries of every row of a pool's page table


class Pool:
    """A pool of pages with the batch arrays of `lens` cached and `news` new
    tokens a sequence.  Every byte that no token's place covers is 0xff (NaN
    scales), so that whatever reads past a sequence shows."""

    def __init__(self, heads, kv_heads, dim, page, lens, news, seed=0, spare=3, extra_rows=0, max_pages=None):
        from hf_llm_b200 import paged
        self.H, self.KV, self.D, self.P, self.lens, self.news = heads, kv_heads, dim, page, list(lens), list(news)
        rng = np.random.default_rng(seed)
        need = [(l + page - 1) // page for l in lens]
        self.max_pages = max_pages or max(1, max(need)) + MORE_PAGES
        self.n_pages = sum(need) + spare
        perm = rng.permutation(self.n_pages)
        table = np.full((len(lens), self.max_pages), -7, np.int32)  # unused entries are no pages
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = perm[at:at + n]
            at += n
        self.table = table
        self.T = sum(news)
        self.rows = self.T + extra_rows
        self.q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.pages = np.full((self.n_pages, kv_heads, page // 16, 18 * dim), 0xff, np.uint8)
        self.cfg = paged.kv_config(heads, kv_heads, dim, Q4_0, page, self.n_pages, self.max_pages)
        self.dev = {}

    def pos(self):
        return np.concatenate([np.arange(l - n, l) for l, n in zip(self.lens, self.news)] + [np.zeros(0, int)]).astype(int)

    def seq(self):
        return np.repeat(np.arange(len(self.lens)), self.news)

    def fill(self, seed=1, spread=1.0):
        """Random codes and scales in every token's place; the f64 keys and values [len, KV, D] of each sequence."""
        rng = np.random.default_rng(seed)
        KV, D, P = self.KV, self.D, self.P
        ks, vs = [], []
        for s, l in enumerate(self.lens):
            kv = []
            for _ in range(2):
                code = rng.integers(0, 16, (l, KV, D)).astype(np.uint8)
                sc = (spread * rng.uniform(0.1, 0.3, (l, KV, D // 32)) * rng.choice([-1, 1], (l, KV, D // 32))).astype(np.float16)
                kv.append((code, sc))
            for b in range((l + 15) // 16):
                n = min(16, l - 16 * b)
                for h in range(KV):
                    part = []
                    for code, sc in kv:
                        c = np.full((16, D), 15, np.uint8)
                        d = np.full((16, D // 32), 0xffff, np.uint16).view(np.float16).copy()
                        c[:n], d[:n] = code[16 * b:16 * b + n, h], sc[16 * b:16 * b + n, h]
                        part += [c, d]
                    self.pages[self.table[s, 16 * b // P], h, 16 * b % P // 16] = block_bytes(*part)
            ks.append(values(*kv[0]))
            vs.append(values(*kv[1]))
        return ks, vs

    def largest_scale(self):
        """Of the values' f16 scales."""
        sc = np.ascontiguousarray(self.pages[..., 17 * self.D:]).view(np.float16).astype(np.float64)
        return float(np.abs(sc[np.isfinite(sc)]).max(initial=0.0))

    def upload(self):
        d = self.dev
        d["q_start"] = torch.from_numpy(self.q_start).cuda()
        d["kv_len"] = torch.tensor(self.lens, dtype=torch.int32).cuda()
        d["table"] = torch.from_numpy(self.table).cuda()
        d["pages"] = torch.from_numpy(self.pages).cuda()
        return self

    def batch(self, max_new=None):
        from hf_llm_b200 import paged
        d = self.dev
        return paged.kv_batch(len(self.lens), self.rows, max(self.news) if max_new is None else max_new,
                              d["q_start"].data_ptr(), d["kv_len"].data_ptr(), d["table"].data_ptr())


def attend(q, ks, vs, news, scale, t_out, e_score, e_prob, tiny=0.0):
    """f64 attention of q [T, H, D] (f64) and a bound of each output's error.

    With scores off by at most e = e_score * scale * max_j sum_d |q_d k_jd| + 2^-20 (the two
    roundings of the exponent's argument and the exponential's own error, a few 2^-22 each, at scores
    below 8 in magnitude from the maximum's; larger ones weigh less), weights are off by a factor 1 +- 2e and the
    normalised sum by 2 * 2e * sum_j p_j |v_j|; probabilities rounded by e_prob relative add
    e_prob * sum_j p_j |v_j|, f32 sums over l keys with one rounding per 16 keys add
    (l / 16 + 16) 2^-24 of it, and the output's rounding half_eps(t_out) of the value.  `tiny` is
    what a term may lose beside that, whatever its size (below f16's smallest step)."""
    outs, bounds = [], []
    a = 0
    for n, k, v in zip(news, ks, vs):
        l, KV, D = k.shape
        H = q.shape[1]
        kk = torch.from_numpy(np.ascontiguousarray(np.repeat(k, H // KV, 1)))
        vv = torch.from_numpy(np.ascontiguousarray(np.repeat(v, H // KV, 1)))
        qq = q[a:a + n]
        a += n
        if n == 0:
            continue
        s = torch.einsum("nhd,lhd->hnl", qq, kk) * scale
        mag = torch.einsum("nhd,lhd->hnl", qq.abs(), kk.abs()) * scale
        hide = torch.arange(l)[None, :] > torch.arange(n)[:, None] + l - n
        s = s.masked_fill(hide, -math.inf)
        m = s.amax(-1, keepdim=True) if l else s.new_zeros(H, n, 1)
        w = torch.where(hide, 0.0, torch.exp(s - torch.where(m == -math.inf, 0.0, m)))
        tot = w.sum(-1, keepdim=True)
        p = w / torch.where(tot == 0, 1.0, tot)
        o = torch.einsum("hnl,lhd->nhd", p, vv)
        wa = torch.einsum("hnl,lhd->nhd", p, vv.abs())
        e = (e_score * mag.masked_fill(hide, 0.0).amax(-1) if l else s.new_zeros(H, n)) + 2.0 ** -20
        e = e.T[..., None]
        outs.append(o)
        bounds.append((4 * e + e_prob + (l / 16 + 16) * 2.0 ** -24) * wa + half_eps(t_out) * o.abs() + l * tiny + 1e-30)
    if not outs:
        return torch.zeros(0, q.shape[1], q.shape[2], dtype=torch.float64), None
    return torch.cat(outs), torch.cat(bounds)


def check_close(got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"error {off.max().item():.3g} is {worst:.3g} times its bound"
    return worst
