"""What the paged K/V cache and attention entry points refuse, without a GPU:
every bad argument gives its status before anything of the device is
touched (the engine handle is a block of zeros)."""
from __future__ import annotations

import ctypes as C

import pytest

F32, F16, Q4_0, Q8_0, BF16 = 0, 1, 2, 8, 30
P = 1 << 20  # stands for an aligned device address: never followed


@pytest.fixture(scope="module")
def calls(pkg):
    from hf_llm_b200 import build
    build.build()
    from hf_llm_b200 import _lib, paged
    L = _lib.lib()
    fake = C.create_string_buffer(1 << 16)
    eng = C.cast(fake, C.c_void_p)

    def cfg(**kw):
        a = dict(n_heads=8, n_kv_heads=2, head_dim=128, kv_type=Q4_0, page_tokens=64, n_pages=10, max_pages=4)
        return paged.kv_config(*{**a, **kw}.values())

    def batch(**kw):
        a = dict(n_seqs=2, n_tokens=3, max_new=2, q_start=P, kv_len=P, page_table=P)
        return paged.kv_batch(*{**a, **kw}.values())

    def append(c=None, b=None, rope=None, x=F32, q=P, qs=1024, k=P, ks=256, v=P, vs=256, pages=P, qo=P, ot=F32, e=eng):
        return L.b2q_kv_append_dev(e, c or cfg(), b or batch(), rope, x, q, qs, k, ks, v, vs, pages, qo, ot, None)

    def gather(c=None, b=None, pages=P, k=P, v=P, ot=F32, e=eng):
        return L.b2q_kv_gather_dev(e, c or cfg(), b or batch(), pages, k, v, ot, None)

    def attn(c=None, b=None, q=P, qt=F32, qs=1024, pages=P, scale=0.1, out=P, ot=F32, work=P, wb=1 << 40, e=eng):
        return L.b2q_attn_paged_dev(e, c or cfg(), b or batch(), q, qt, qs, pages, scale, out, ot, work, wb, None)

    def prompt(e=eng, q=P, qs=1024, k=P, ks=256, v=P, vs=256, scale=0.1, out=P, **kw):
        a = dict(n_heads=8, n_kv_heads=2, head_dim=128, type=F16, n_seqs=2, n_q=3, n_kv=3, max_new=2, q_start=P, kv_start=P)
        return L.b2q_attn_prompt_dev(e, paged.prompt(*{**a, **kw}.values()), q, qs, k, ks, v, vs, scale, out, None)

    return dict(cfg=cfg, batch=batch, append=append, gather=gather, attn=attn, prompt=prompt, lib=L, m=_lib, paged=paged, keep=fake)


BAD_CFG = [(dict(n_heads=0), 1), (dict(n_kv_heads=0), 1), (dict(n_heads=7), 1), (dict(n_heads=2048), 1), (dict(head_dim=96), 6),
           (dict(head_dim=256), 6), (dict(kv_type=F16), 6), (dict(kv_type=Q8_0), 6), (dict(page_tokens=0), 1),
           (dict(page_tokens=24), 1), (dict(page_tokens=8192), 1), (dict(page_tokens=-16), 1), (dict(n_pages=0), 1),
           (dict(max_pages=0), 1), (dict(max_pages=1 << 25), 1), (dict(n_heads=-8), 1)]


@pytest.mark.parametrize("bad,status", BAD_CFG)
def test_bad_configurations(calls, bad, status):
    c = calls["cfg"](**bad)
    for f in ("append", "gather", "attn"):
        assert calls[f](c=c) == status, f
        assert calls["lib"].b2q_last_error()
    assert calls["lib"].b2q_kv_page_bytes(c) == 0
    with pytest.raises(calls["m"].B2QError):
        calls["paged"].page_bytes(c)


@pytest.mark.parametrize("bad", [dict(n_seqs=-1), dict(n_tokens=-1), dict(max_new=-1), dict(n_seqs=65536), dict(q_start=None),
                                 dict(kv_len=None), dict(page_table=None)])
def test_bad_batches(calls, bad):
    for f in ("append", "gather", "attn"):
        assert calls[f](b=calls["batch"](**bad)) == 1, f


@pytest.mark.parametrize("bad,status", [
    (dict(e=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(pages=None), 1), (dict(pages=P + 8), 1), (dict(qo=None), 1),
    (dict(k=P + 4), 1), (dict(q=P + 8), 1), (dict(ks=128), 1), (dict(qs=1023), 1), (dict(vs=257), 1), (dict(x=Q4_0), 6), (dict(ot=Q8_0), 6),
    (dict(qs=1 << 33), 1), (dict(qs=-1024), 1)])
def test_bad_appends(calls, bad, status):
    assert calls["append"](**bad) == status


@pytest.mark.parametrize("args", [(132, 5, P, P), (12, 5, P, P), (-8, 5, P, P), (64, 0, P, P), (64, 5, 0, P), (64, 5, P, P + 4)])
def test_bad_rotations(calls, args):
    assert calls["append"](rope=calls["paged"].rope(*args)) == 1


@pytest.mark.parametrize("bad,status", [(dict(e=None), 1), (dict(pages=None), 1), (dict(k=None, v=None), 1), (dict(k=P + 2), 1),
                                        (dict(v=P + 8), 1), (dict(ot=Q4_0), 6)])
def test_bad_gathers(calls, bad, status):
    assert calls["gather"](**bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(e=None), 1), (dict(q=None), 1), (dict(q=P + 4), 1), (dict(qs=1000), 1), (dict(pages=None), 1), (dict(pages=P + 1), 1),
    (dict(out=None), 1), (dict(out=P + 8), 1), (dict(qt=Q4_0), 6), (dict(ot=Q8_0), 6), (dict(scale=0.0), 1), (dict(scale=-1.0), 1),
    (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(scale=2e30), 1), (dict(work=None), 1), (dict(work=P + 8), 1), (dict(wb=0), 1)])
def test_bad_attention(calls, bad, status):
    assert calls["attn"](**bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(e=None), 1), (dict(n_heads=7), 1), (dict(n_kv_heads=-2), 1), (dict(head_dim=256), 6), (dict(type=F32), 6), (dict(type=Q4_0), 6),
    (dict(n_seqs=-1), 1), (dict(n_q=-1), 1), (dict(n_kv=-1), 1), (dict(max_new=-1), 1), (dict(n_seqs=70000), 1), (dict(q_start=None), 1),
    (dict(kv_start=None), 1), (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(q=P + 2), 1),
    (dict(ks=255), 1), (dict(vs=250), 1), (dict(qs=512), 1), (dict(scale=0.0), 1), (dict(scale=2e30), 1), (dict(scale=float("nan")), 1)])
def test_bad_prompts(calls, bad, status):
    assert calls["prompt"](**bad) == status


def test_empty_batches_do_nothing(calls):
    for f in ("append", "gather", "attn"):
        assert calls[f](b=calls["batch"](n_tokens=0)) == 0
        assert calls[f](b=calls["batch"](n_seqs=0)) == 0
    assert calls["prompt"](n_q=0) == 0 and calls["prompt"](n_seqs=0) == 0


def test_page_bytes(calls):
    assert calls["paged"].page_bytes(calls["cfg"]()) == 2 * 4 * 18 * 128
    assert calls["paged"].page_bytes(calls["cfg"](head_dim=64, page_tokens=16, n_kv_heads=8)) == 8 * 18 * 64


def test_workspace_of_bad_arguments(calls):
    """0, and a text of its own rather than the last failure's."""
    work = calls["lib"].b2q_attn_paged_work_bytes
    for e, c, b, text in ((None, calls["cfg"](), calls["batch"](), "engine"), (calls["keep"], calls["cfg"](n_heads=7), calls["batch"](), "heads"),
                          (calls["keep"], calls["cfg"](), calls["batch"](kv_len=None), "NULL array")):
        assert calls["prompt"](type=Q4_0) == 6  # another failure first
        assert work(e and C.cast(e, C.c_void_p), c, b) == 0
        said = calls["lib"].b2q_last_error().decode()
        assert "b2q_attn_paged_work_bytes" in said and text in said
    assert work(C.cast(calls["keep"], C.c_void_p), calls["cfg"](), calls["batch"]()) > 0
