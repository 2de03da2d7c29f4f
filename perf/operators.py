"""Cases of the operators that serve many sequences at once from a paged 4-bit K/V cache.

Four operators, one "op" each:

* append -- rotate the new tokens' queries and keys by their positions and write keys and
            values into the pages, 32 values to a block of 4-bit codes and one f16 scale;
* gather -- read rows of the cache back as numbers;
* paged  -- attention of the newest tokens of every sequence over its cached keys and values;
* prompt -- causal attention over packed prompts, of f16 or bf16 queries, keys and values.

`run` computes them with elementary torch operations, or, where `own` is true, through the
calls a user makes of the package.

A cached block is 16 consecutive tokens of one K/V head, 18 * D bytes: the keys' codes, the
keys' scales [16][D / 32] f16, the values' codes, the values' scales.  A code is value / scale + 8 in
0..15.  Keys: token row of D / 2 bytes, [4 lanes][D / 32 blocks] words, eight consecutive
dims 32 b + 8 t + n in nibble n.  Values: [8 dims mod 8][token pair][token of the pair] pieces
of D / 16 bytes in two halves of 8 tokens; nibble j is dim 8 j + g.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
Q4_0 = 2
THETA = 500000.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one user, one token, the benchmark's context after its 512-token prompt: latency
        {"name": "paged one 585", "op": "paged", "seqs": 1, "kv": 585, "ragged": False, "new": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "q": "f32", "out": "f32"},
        # one user with a very long conversation: the whole GPU on one sequence
        {"name": "paged one 131072", "op": "paged", "seqs": 1, "kv": 131072, "ragged": False, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 256, "q": "f32", "out": "f32"},
        # a full batch of users at very different points of their conversations
        {"name": "paged 64 ragged", "op": "paged", "seqs": 64, "kv": 8192, "ragged": True, "new": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "q": "f16", "out": "f16"},
        # checking drafted tokens: five queries a sequence, eight query heads to a K/V head, small pages
        {"name": "paged 16 drafted", "op": "paged", "seqs": 16, "kv": 4001, "ragged": True, "new": 5, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 16, "q": "bf16", "out": "bf16"},
        # the benchmark's prompt
        {"name": "prompt 512", "op": "prompt", "seqs": 1, "new": 512, "prefix": 0, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "f16"},
        # prompts of different users packed one behind the other
        {"name": "prompt 16 ragged", "op": "prompt", "seqs": 16, "new": 1800, "prefix": 0, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "bf16"},
        # a prompt as long as the model's context, 70B-shaped heads
        {"name": "prompt 8192", "op": "prompt", "seqs": 1, "new": 8192, "prefix": 0, "ragged": False, "heads": 64, "kv_heads": 8,
         "dim": 128, "type": "bf16"},
        # the next piece of prompts whose first part is in the cache already; 64-wide heads
        {"name": "prompt 6 behind 2000", "op": "prompt", "seqs": 6, "new": 301, "prefix": 2000, "ragged": True, "heads": 16,
         "kv_heads": 4, "dim": 64, "type": "f16"},
        # one decode step of a batch: a new token for every sequence
        {"name": "append 64 x 1", "op": "append", "seqs": 64, "new": 1, "kv": 2048, "ragged": True, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "x": "f32", "out": "f16"},
        # a whole prompt's keys and values
        {"name": "append 8192", "op": "append", "seqs": 1, "new": 8192, "kv": 8192, "ragged": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "x": "f32", "out": "bf16"},
        # the cached part of four prompts, read back for the attention of what follows it
        {"name": "gather 4 x 8192", "op": "gather", "seqs": 4, "new": 8192, "kv": 8192, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "out": "f16"},
        # a short shared beginning, read back exactly
        {"name": "gather 333", "op": "gather", "seqs": 1, "new": 333, "kv": 333, "ragged": False, "heads": 8, "kv_heads": 2,
         "dim": 64, "page": 32, "out": "f32"},
    ]


HEADS = [(32, 8, 128), (64, 8, 128), (8, 2, 128), (16, 16, 128), (16, 4, 64), (24, 8, 128), (8, 1, 64), (32, 4, 128), (40, 8, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["paged", "paged", "prompt", "prompt", "append", "gather"])
    heads, kv_heads, dim = rng.choice(HEADS)
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "ragged": rng.random() < 0.7}
    if op == "prompt":
        c["type"] = rng.choice(["f16", "bf16"])
        c["new"] = _log(rng, 2, 6000)
        c["prefix"] = _log(rng, 1, 4000) if rng.random() < 0.4 else 0
        # the score matrices of the plain form, and the work, stay under the largest listed case's
        cost = heads * c["new"] * (c["new"] + c["prefix"])
        c["seqs"] = _log(rng, 1, max(1, min(48, int(3.5e9 / cost))))
        return c
    c["page"] = rng.choice([16, 32, 48, 64, 128, 256])
    if op == "paged":
        c["new"] = rng.choice([1, 1, 1, 2, 3, 5, 8])
        c["seqs"] = _log(rng, 1, 200)
        c["kv"] = _log(rng, c["new"], max(c["new"], min(131072, int(4.0e8 / (c["seqs"] * kv_heads * dim)))))
        c["q"] = rng.choice(["f32", "f16", "bf16"])
        c["out"] = rng.choice([c["q"], c["q"], "f32"])
        return c
    c["seqs"] = _log(rng, 1, 100)
    c["new"] = _log(rng, 1, max(1, 8192 * 4096 // (c["seqs"] * heads * dim)))
    c["kv"] = c["new"] if op == "gather" else c["new"] + _log(rng, 1, 4000)
    c["out"] = rng.choice(["f32", "f16", "bf16"])
    if op == "append":
        c["x"] = rng.choice(["f32", "f16", "bf16"])
    return c


def _lens(case):
    """(new tokens, cached tokens with them) of every sequence: a function of the case alone."""
    n, new = case["seqs"], case["new"]
    r = random.Random(n * 1000003 + new * 7919 + case.get("kv", 0) + case.get("prefix", 0))
    if case["op"] == "prompt":
        ns = [new if not case["ragged"] else r.randint(max(1, new // 8), new) for _ in range(n)]
        ps = [case["prefix"] if not case["ragged"] else r.randint(0, case["prefix"]) for _ in range(n)]
        ns[-1], ps[0] = new, case["prefix"]
        return ns, [a + b for a, b in zip(ns, ps)]
    if case["op"] == "gather":
        ns = [new if not case["ragged"] else r.randint(max(1, new // 8), new) for _ in range(n)]
        ns[0] = new
        return ns, list(ns)
    # one query token or the same number of drafted ones for each; the longest cache is the case's
    ls = [case["kv"] if not case["ragged"] else r.randint(new, case["kv"]) for _ in range(n)]
    ls[-1] = case["kv"]
    return [new] * n, ls


def work(case):
    ns, ls = _lens(case)
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    row4 = KV * 2 * (D // 2 + D // 16)  # cached bytes of a token, keys and values
    if case["op"] == "prompt":
        pairs = sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(ns, ls))
        return {"bytes": 2 * D * (2 * H * sum(ns) + 2 * KV * sum(ls)), "flops": 4 * H * D * pairs}
    if case["op"] == "paged":
        pairs = sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(ns, ls))
        return {"bytes": sum(ls) * row4 + sum(ns) * H * D * (size[case["q"]] + size[case["out"]]), "flops": 4 * H * D * pairs}
    T = sum(ns)
    if case["op"] == "append":  # and the new rows read back
        return {"bytes": T * (size[case["x"]] * (H + 2 * KV) * D + size[case["out"]] * H * D + 2 * row4 + 2 * 4 * KV * D + 4 * D),
                "flops": 3 * T * (H + KV) * D + 4 * T * KV * D}
    return {"bytes": T * (row4 + 2 * size[case["out"]] * KV * D), "flops": 2 * T * KV * D}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    ns, ls = _lens(case)
    B, T, i32 = len(ns), sum(ns), torch.int32
    dev = {"device": "cuda"}

    def randn(*shape):
        return torch.randn(*shape, generator=g, **dev)

    def cum(v):
        return torch.tensor([0] + v, dtype=torch.int64).cumsum(0).to(i32).cuda()

    s = {"case": dict(case), "q_start": cum(ns), "n_tokens": T, "max_new": max(ns), "max_kv": max(ls)}
    if case["op"] == "prompt":
        t = TYPES[case["type"]]
        s["kv_start"] = cum(ls)
        s["q"] = randn(T, H, D).to(t)
        s["k"] = randn(sum(ls), KV, D).to(t)
        s["v"] = randn(sum(ls), KV, D).to(t)
        s["out"] = torch.empty(T, H, D, dtype=t, **dev)
        return s
    P = case["page"]
    need = [(l + P - 1) // P for l in ls]
    s["max_pages"], s["n_pages"] = max(need), sum(need) + 3
    perm = torch.randperm(s["n_pages"], generator=g, **dev)  # a sequence's pages lie anywhere in the pool
    # entry (sequence, i) of the table is page first[sequence] + i of the permutation
    at = cum(need)[:-1].long()[:, None] + torch.arange(s["max_pages"], **dev)[None, :]
    s["page_table"] = perm[at.clamp(max=s["n_pages"] - 1)].to(i32).contiguous()
    s["kv_len"] = torch.tensor(ls, dtype=i32).cuda()
    if case["op"] == "append":
        x = TYPES[case["x"]]
        s["q"], s["k"], s["v"] = randn(T, H, D).to(x), randn(T, KV, D).to(x), randn(T, KV, D).to(x)
        s["pages"] = torch.zeros(s["n_pages"], KV, P // 16, 18 * D, dtype=torch.uint8, **dev)
        ang = torch.arange(max(ls), dtype=torch.float64, **dev)[:, None] * (
            THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, **dev) / D))[None, :]
        s["cos"], s["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
        s["q_out"] = torch.empty(T, H, D, dtype=TYPES[case["out"]], **dev)
        s["k_out"] = torch.empty(T, KV, D, **dev)
        s["v_out"] = torch.empty(T, KV, D, **dev)
        return s
    # cached blocks: any codes, scales as 4-bit blocks of values of unit spread have them, of either sign
    pages = torch.randint(0, 256, (s["n_pages"], KV, P // 16, 18 * D), dtype=torch.uint8, generator=g, **dev)
    for o in (8 * D, 17 * D):
        sc = (0.15 + 0.15 * torch.rand(*pages.shape[:3], D // 2, generator=g, **dev))
        sc = sc * (1 - 2 * torch.randint(0, 2, sc.shape, generator=g, **dev))
        pages[..., o:o + D] = sc.half().view(torch.uint8)
    s["pages"] = pages
    if case["op"] == "gather":
        t = TYPES[case["out"]]
        s["k_out"] = torch.empty(T, KV, D, dtype=t, **dev)
        s["v_out"] = torch.empty(T, KV, D, dtype=t, **dev)
        return s
    s["q"] = randn(T, H, D).to(TYPES[case["q"]])
    s["out"] = torch.empty(T, H, D, dtype=TYPES[case["out"]], **dev)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _values(blocks, D):
    """Keys and values [..., 16, D] in f32 of cached blocks [..., 18 * D] of bytes."""
    lead = blocks.shape[:-1]
    k = _nibbles(blocks[..., :8 * D]).view(*lead, 16, 4, D // 32, 8).transpose(-2, -3).reshape(*lead, 16, D // 32, 32)
    v = _nibbles(blocks[..., 9 * D:17 * D]).view(*lead, 2, 8, 4, 2, D // 8)
    v = v.movedim(-4, -1).reshape(*lead, 16, D // 32, 32)
    ks = blocks[..., 8 * D:9 * D].contiguous().view(torch.float16).view(*lead, 16, D // 32, 1).float()
    vs = blocks[..., 17 * D:].contiguous().view(torch.float16).view(*lead, 16, D // 32, 1).float()
    return ((k.float() - 8) * ks).flatten(-2), ((v.float() - 8) * vs).flatten(-2)


def _cached(s):
    """Keys and values [sequences, positions, K/V heads, D] of the sequences' pages."""
    D = s["case"]["dim"]
    k, v = _values(s["pages"][s["page_table"].long()].transpose(2, 3).flatten(1, 2), D)
    return k.transpose(2, 3).flatten(1, 2), v.transpose(2, 3).flatten(1, 2)


def _tokens(s, start):
    """Sequence and place in it of every packed token."""
    n = (start[1:] - start[:-1]).long()
    at = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=int(s["n_tokens"]) if start is s["q_start"] else None)
    return at, torch.arange(at.numel(), device="cuda") - start[:-1].long()[at]


def _attend(q, k, v, seen):
    """softmax(q k / sqrt(D)) v of q [B, KV, G, R, D], k and v [B, KV, L, D], over the first seen [B, R] keys."""
    B, KV, G, R, D = q.shape
    sc = torch.matmul(q.reshape(B, KV, G * R, D) * (1 / math.sqrt(D)), k.transpose(2, 3)).view(B, KV, G, R, -1)
    hidden = torch.arange(k.shape[2], device="cuda")[None, None, :] >= seen[:, :, None]
    sc.masked_fill_(hidden[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    sc.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    tot = sc.sum(-1, keepdim=True)
    o = torch.matmul(sc.view(B, KV, G * R, -1), v).view(B, KV, G, R, D)
    return o / torch.where(tot == 0, torch.ones_like(tot), tot)


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _to4(x):
    """The values that blocks of 4-bit codes hold for x [..., D]: scale = (the first value of the largest magnitude) / -8 in f16."""
    b = x.unflatten(-1, (-1, 32))
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = (big / -8).clamp(-65504, 65504).half().float()
    code = (torch.where(d == 0, torch.zeros_like(b), b / d).round() + 8).clamp(0, 15)
    return ((code - 8) * d).flatten(-2)


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    KV, D = c["kv_heads"], c["dim"]
    if c["op"] == "append":
        seq, at = _tokens(s, s["q_start"])
        n = (s["q_start"][1:] - s["q_start"][:-1]).long()
        pos = (s["kv_len"].long() - n)[seq] + at
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        return {"q": _rotate(s["q"], cos, sin).to(TYPES[c["out"]]), "k": _to4(_rotate(s["k"], cos, sin)), "v": _to4(s["v"].float())}
    if c["op"] == "gather":
        k, v = _cached(s)
        seq, at = _tokens(s, s["q_start"])
        pos = (s["kv_len"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long())[seq] + at
        return {"k": k[seq, pos].to(TYPES[c["out"]]), "v": v[seq, pos].to(TYPES[c["out"]])}
    B, G, R = c["seqs"], c["heads"] // KV, s["max_new"]
    seq, at = _tokens(s, s["q_start"])
    q = torch.zeros(B, R, c["heads"], D, device="cuda")
    q[seq, at] = s["q"].float()
    if c["op"] == "paged":
        k, v = (x.transpose(1, 2) for x in _cached(s))
        lens = s["kv_len"].long()
        to = TYPES[c["out"]]
    else:
        lens = (s["kv_start"][1:] - s["kv_start"][:-1]).long()
        kseq, kat = _tokens(s, s["kv_start"])
        k = torch.zeros(B, s["max_kv"], KV, D, device="cuda")
        v = torch.zeros(B, s["max_kv"], KV, D, device="cuda")
        k[kseq, kat], v[kseq, kat] = s["k"].float(), s["v"].float()
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        to = TYPES[c["type"]]
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    seen = lens[:, None] - n[:, None] + torch.arange(R, device="cuda")[None, :] + 1
    o = _attend(q.view(B, R, KV, G, D).permute(0, 2, 3, 1, 4), k, v, seen)
    return o.permute(0, 3, 1, 2, 4).reshape(B, R, c["heads"], D)[seq, at].to(to)


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _package():
    name = "hf_llm_b200"
    if name not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "huggingface-local-llm-ui_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    from hf_llm_b200 import paged
    from hf_llm_b200.engine import CudaEngine
    return paged, CudaEngine.global_(torch.cuda.current_device())


def _run_own(s):
    paged, eng = _package()
    c = s["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["dim"]
    stream = torch.cuda.current_stream().cuda_stream or 1  # 1: cudaStreamLegacy, torch's default stream
    if c["op"] == "prompt":
        eng.attn_prompt_dev(
            paged.prompt(H, KV, D, GGML[c["type"]], c["seqs"], s["n_tokens"], s["k"].shape[0], s["max_new"], s["q_start"].data_ptr(),
                         s["kv_start"].data_ptr()),
            s["q"].data_ptr(), H * D, s["k"].data_ptr(), KV * D, s["v"].data_ptr(), KV * D, 1 / math.sqrt(D), s["out"].data_ptr(), stream)
        return s["out"]
    cfg = paged.kv_config(H, KV, D, Q4_0, c["page"], s["n_pages"], s["max_pages"])
    batch = paged.kv_batch(c["seqs"], s["n_tokens"], s["max_new"], s["q_start"].data_ptr(), s["kv_len"].data_ptr(),
                           s["page_table"].data_ptr())
    if c["op"] == "paged":
        if "work" not in s:  # a program keeps one for each stream
            s["work"] = torch.empty(eng.attn_paged_work_bytes(cfg, batch), dtype=torch.uint8, device="cuda")
        eng.attn_paged_dev(cfg, batch, s["q"].data_ptr(), GGML[c["q"]], H * D, s["pages"].data_ptr(), 1 / math.sqrt(D),
                           s["out"].data_ptr(), GGML[c["out"]], s["work"].data_ptr(), s["work"].numel(), stream)
        return s["out"]
    if c["op"] == "append":
        rope = paged.rope(D, s["cos"].shape[0], s["cos"].data_ptr(), s["sin"].data_ptr())
        eng.kv_append_dev(cfg, batch, rope, GGML[c["x"]], s["q"].data_ptr(), H * D, s["k"].data_ptr(), KV * D, s["v"].data_ptr(), KV * D,
                          s["pages"].data_ptr(), s["q_out"].data_ptr(), GGML[c["out"]], stream)
        eng.kv_gather_dev(cfg, batch, s["pages"].data_ptr(), s["k_out"].data_ptr(), s["v_out"].data_ptr(), GGML["f32"], stream)
        return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
    eng.kv_gather_dev(cfg, batch, s["pages"].data_ptr(), s["k_out"].data_ptr(), s["v_out"].data_ptr(), GGML[c["out"]], stream)
    return {"k": s["k_out"], "v": s["v_out"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _rows64(s, b, length):
    """Keys and values [length, KV, D] in f64 of sequence b, nibble by nibble from the block's description."""
    c = s["case"]
    KV, D, P = c["kv_heads"], c["dim"], c["page"]
    pos = torch.arange(length, device="cuda")
    base = s["page_table"][b].long()[pos // P] * (KV * (P // 16)) + (pos % P) // 16
    base = (base[:, None] + torch.arange(KV, device="cuda")[None, :] * (P // 16)) * (18 * D)  # the block's first byte
    raw = s["pages"].view(-1)
    tok = (pos % 16)[:, None, None]
    dim = torch.arange(D, device="cuda")[None, None, :]
    base = base[:, :, None]
    byte_k = tok * (D // 2) + (dim % 32) // 8 * (D // 8) + dim // 32 * 4 + dim % 8 // 2
    byte_v = tok // 8 * (4 * D) + dim % 8 * (D // 2) + tok % 8 // 2 * (D // 8) + tok % 2 * (D // 16) + dim // 8 // 2

    def scale(off):
        lo = raw[base + off + (tok * (D // 32) + dim // 32) * 2].to(torch.int32)
        hi = raw[base + off + (tok * (D // 32) + dim // 32) * 2 + 1].to(torch.int32)
        return (lo | hi << 8).to(torch.int16).view(torch.float16).double()

    code_k = raw[base + byte_k].long() >> (dim % 2 * 4) & 15
    code_v = raw[base + 9 * D + byte_v].long() >> (dim // 8 % 2 * 4) & 15
    return (code_k - 8).double() * scale(8 * D), (code_v - 8).double() * scale(17 * D)


def exact(case, seed):
    s = prepare(case, seed)
    ns, ls = _lens(case)
    H, KV, D = case["heads"], case["kv_heads"], case["dim"]
    G = H // KV
    if case["op"] == "append":
        pos = torch.cat([torch.arange(l - n, l, device="cuda") for n, l in zip(ns, ls)])
        c, sn = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
        q = s["q"].double()
        a, b = q[..., :D // 2], q[..., D // 2:]
        # what a block of 4-bit codes holds hangs on roundings: it has no value in 64 bits
        return {"q": torch.cat((a * c - b * sn, a * sn + b * c), -1), "k": None, "v": None}
    if case["op"] == "gather":
        ks, vs = zip(*(_rows64(s, b, ls[b]) for b in range(case["seqs"])))
        return {"k": torch.cat(ks), "v": torch.cat(vs)}
    out, qa, ka = [], 0, 0
    for b, (n, l) in enumerate(zip(ns, ls)):
        q = s["q"][qa:qa + n].double()
        if case["op"] == "paged":
            k, v = _rows64(s, b, l)
        else:
            k, v = s["k"][ka:ka + l].double(), s["v"][ka:ka + l].double()
        qa, ka = qa + n, ka + l
        hide = torch.ones(n, l, device="cuda", dtype=torch.bool).tril(l - n).logical_not()
        heads = []
        for h in range(H):
            w = (q[:, h] @ k[:, h // G].T) / math.sqrt(D)
            heads.append(torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v[:, h // G])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
