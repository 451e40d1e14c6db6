"""Refusals of the paged-cache entry points and what their bindings assume: no kernel runs here."""
import ctypes as C

import numpy as np
import pytest
import torch

import paged_ref as R
from fblt_b200 import lib as L

P = 1 << 20  # an aligned address that is never read: every call below is refused, or has nothing to do


def cache(**kw):
    c = L.PagedCache()
    c.format, c.num_kv_heads, c.head_dim, c.page_size, c.num_pages, c.max_pages = L.KV_E4M3, 2, 64, 16, 8, 4
    c.k_codes = c.v_codes = c.k_exp = c.v_exp = c.page_table = P
    c.page_table_stride = 4
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append(**kw):
    d = L.PagedAppendDesc()
    ck = {k[6:]: kw.pop(k) for k in list(kw) if k.startswith("cache_")}
    d.cache, d.batch, d.num_heads, d.total_rows = cache(**ck), 2, 4, 3
    d.cu_new = d.base_len = d.k = d.v = d.q = d.q_out = P
    d.k_stride = d.v_stride = 128
    d.q_stride = d.q_out_stride = 256
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def read(**kw):
    d = L.PagedReadDesc()
    ck = {k[6:]: kw.pop(k) for k in list(kw) if k.startswith("cache_")}
    d.cache, d.batch, d.total_rows = cache(**ck), 2, 3
    d.cu_rows = d.k_out = d.v_out = P
    d.k_out_stride = d.v_out_stride = 128
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def attn(**kw):
    d = L.PagedAttnDesc()
    ck = {k[6:]: kw.pop(k) for k in list(kw) if k.startswith("cache_")}
    d.cache, d.batch, d.num_heads, d.total_rows, d.max_new, d.max_len = cache(**ck), 2, 4, 3, 2, 64
    d.cu_new = d.base_len = d.q = d.out = P
    d.q_stride = d.out_stride = 256
    d.scale = 0.125
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def norm(**kw):
    d = L.QkNormRopeDesc()
    d.rows, d.num_heads, d.num_kv_heads, d.head_dim, d.rope_len = 3, 4, 2, 64, 8
    d.q = d.k = d.q_out = d.k_out = d.q_gain = d.k_gain = d.rope_cos = d.rope_sin = d.pos = P
    d.q_stride = d.q_out_stride = 256
    d.k_stride = d.k_out_stride = 128
    d.eps = 1e-6
    for k, v in kw.items():
        setattr(d, k, v)
    return d


CACHE_BAD = [(dict(format=2), L.ERR_ARG), (dict(head_dim=48), L.ERR_UNSUPPORTED), (dict(head_dim=0), L.ERR_UNSUPPORTED),
             (dict(num_kv_heads=0), L.ERR_ARG), (dict(page_size=8), L.ERR_UNSUPPORTED), (dict(page_size=24), L.ERR_UNSUPPORTED),
             (dict(page_size=2048), L.ERR_UNSUPPORTED), (dict(num_pages=-1), L.ERR_ARG), (dict(max_pages=-1), L.ERR_ARG),
             (dict(k_codes=None), L.ERR_ARG), (dict(v_codes=P + 8), L.ERR_ARG), (dict(k_exp=None), L.ERR_ARG),
             (dict(v_exp=P + 1), L.ERR_ARG), (dict(page_table=None), L.ERR_ARG), (dict(page_table=P + 2), L.ERR_ARG),
             (dict(page_table_stride=3), L.ERR_ARG), (dict(status=P + 1), L.ERR_ARG)]


@pytest.mark.parametrize("bad,want", CACHE_BAD)
def test_cache_description_is_checked_everywhere(bad, want):
    lib = L.load()
    bad = {"cache_" + k: v for k, v in bad.items()}
    assert lib.fblt_paged_append(C.byref(append(**bad)), None) == want
    assert lib.fblt_paged_read(C.byref(read(**bad)), None) == want
    assert lib.fblt_paged_attn(C.byref(attn(**bad)), P, 1 << 30, None) == want
    assert lib.fblt_paged_attn_workspace(C.byref(attn(**bad))) == 0


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(total_rows=-1), dict(cu_new=None), dict(base_len=None), dict(k=None), dict(v=None), dict(q=None),
    dict(q_out=None), dict(num_heads=0), dict(k=P + 4), dict(k_stride=127), dict(k_stride=130), dict(v_stride=64),
    dict(q_stride=128), dict(q_out_stride=254), dict(q_gain=P + 4), dict(q_gain=P, eps=-1.0), dict(k_gain=P, eps=float("nan")),
    dict(rope_cos=P), dict(rope_cos=P, rope_sin=P, rope_len=0), dict(rope_cos=P + 4, rope_sin=P, rope_len=4),
    dict(q_out_stride=260)])
def test_append_refuses(bad):
    assert L.load().fblt_paged_append(C.byref(append(**bad)), None) == L.ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(total_rows=-2), dict(cu_rows=None), dict(k_out=None, v_out=None), dict(out_type=2), dict(k_out=P + 4),
    dict(k_out_stride=64), dict(v_out_stride=130), dict(out_type=1, k_out_stride=132)])
def test_read_refuses(bad):
    assert L.load().fblt_paged_read(C.byref(read(**bad)), None) == L.ERR_ARG


@pytest.mark.parametrize("bad,want", [
    (dict(batch=-1), L.ERR_ARG), (dict(max_new=-1), L.ERR_ARG), (dict(max_len=-1), L.ERR_ARG), (dict(num_heads=3), L.ERR_ARG),
    (dict(num_heads=0), L.ERR_ARG), (dict(window=-1), L.ERR_ARG), (dict(splits=-1), L.ERR_ARG), (dict(scale=float("inf")), L.ERR_ARG),
    (dict(scale=float("nan")), L.ERR_ARG), (dict(batch=65536), L.ERR_LIMIT), (dict(cu_new=None), L.ERR_ARG), (dict(q=None), L.ERR_ARG),
    (dict(base_len=None), L.ERR_ARG), (dict(out=None), L.ERR_ARG), (dict(q_stride=255), L.ERR_ARG), (dict(out_stride=258), L.ERR_ARG),
    (dict(q=P + 8), L.ERR_ARG), (dict(max_new=2**30, num_heads=8, q_stride=512, out_stride=512), L.ERR_LIMIT),
    (dict(max_new=2**28), L.ERR_LIMIT)])
def test_attention_refuses(bad, want):
    assert L.load().fblt_paged_attn(C.byref(attn(**bad)), P, 1 << 30, None) == want


@pytest.mark.parametrize("bad,want", [
    (dict(rows=-1), L.ERR_ARG), (dict(head_dim=256), L.ERR_UNSUPPORTED), (dict(q=None), L.ERR_ARG), (dict(k_out=None), L.ERR_ARG),
    (dict(q=None, q_out=None, k=None, k_out=None), L.ERR_ARG), (dict(num_heads=0), L.ERR_ARG), (dict(num_kv_heads=-3), L.ERR_ARG),
    (dict(q_stride=200), L.ERR_ARG), (dict(k_out_stride=129), L.ERR_ARG), (dict(q_out=P + 8), L.ERR_ARG), (dict(k_gain=P + 8), L.ERR_ARG),
    (dict(eps=float("inf")), L.ERR_ARG), (dict(rope_sin=None), L.ERR_ARG), (dict(pos=None), L.ERR_ARG), (dict(rope_len=0), L.ERR_ARG),
    (dict(q_out_stride=512), L.ERR_ARG)])
def test_norm_rope_refuses(bad, want):
    assert L.load().fblt_qk_norm_rope(C.byref(norm(**bad)), None) == want


def test_null_and_empty_calls():
    lib = L.load()
    for f in (lib.fblt_qk_norm_rope, lib.fblt_paged_append, lib.fblt_paged_read, lib.fblt_paged_self_attention_step):
        assert f(None, None) == L.ERR_ARG
    assert lib.fblt_paged_attn(None, None, 0, None) == L.ERR_ARG and lib.fblt_paged_attn_workspace(None) == 0
    empty = dict(cache_k_codes=None, cache_v_codes=None, cache_k_exp=None, cache_v_exp=None, cache_page_table=None)
    assert lib.fblt_paged_append(C.byref(append(batch=0, total_rows=0, **empty)), None) == L.OK
    assert lib.fblt_paged_append(C.byref(append(total_rows=0, k=None, v=None)), None) == L.OK
    assert lib.fblt_paged_read(C.byref(read(total_rows=0)), None) == L.OK
    assert lib.fblt_paged_attn(C.byref(attn(total_rows=0)), None, 0, None) == L.OK
    assert lib.fblt_paged_attn(C.byref(attn(max_new=0)), None, 0, None) == L.OK
    assert lib.fblt_qk_norm_rope(C.byref(norm(rows=0)), None) == L.OK


def test_step_refuses_before_it_launches():
    lib, d = L.load(), L.PagedStepDesc()
    d.cache, d.batch, d.num_heads, d.total_rows, d.max_new, d.max_len = cache(), 2, 4, 3, 2, 64
    d.cu_new = d.base_len = d.input = d.packed_qkv = d.packed_proj = d.output = d.qkv_work = d.combined_work = P
    d.input_stride = d.output_stride = 256
    d.eps = 1e-6
    for name, v in (("input", None), ("output_stride", 128), ("num_heads", 3), ("rope_cos", P), ("qkv_work", P + 4), ("max_new", 0),
                    ("window", -1)):
        keep = getattr(d, name)
        setattr(d, name, v)
        assert lib.fblt_paged_self_attention_step(C.byref(d), None) == L.ERR_ARG, name
        setattr(d, name, keep)


def test_reference_code_values():
    """The test's own table of e4m3 values against torch's type."""
    t = R.code_table("e4m3")
    f = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    fin = np.isfinite(f)
    assert (t[fin] == f[fin]).all() and set(np.flatnonzero(~fin)) == {0x7f, 0xff} and t[0x7f] == 480
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((6, 32)) * 10.0 ** rng.integers(-6, 6, (6, 1))).astype(np.float32).astype(np.float64)
    for fmt in ("e4m3", "int8"):
        c, e = R.quantise(x, fmt)
        y = R.code_table(fmt)[c] * 2.0 ** e.astype(np.float64)[:, None]
        step = 2.0 ** e.astype(np.float64)[:, None]
        bound = np.maximum(np.abs(x) * 2.0 ** -4, step * 2.0 ** -10) if fmt == "e4m3" else step / 2
        assert (np.abs(x - y) <= bound).all()
