"""Refusals of the paged cache's entry points that depend on the launch that a call would make: no kernel runs here."""
import ctypes as C

import pytest

from fblt_b200 import lib as L
from test_paged_host import P, attn, cache


def step(**kw):
    d = L.PagedStepDesc()
    d.cache, d.batch, d.num_heads, d.total_rows, d.max_new, d.max_len = cache(), 2, 4, 3, 2, 64
    d.cu_new = d.base_len = d.input = d.packed_qkv = d.packed_proj = d.output = d.qkv_work = d.combined_work = P
    d.input_stride = d.output_stride = 256
    d.eps = 1e-6
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("bad,want", [
    (dict(workspace=P + 8, workspace_bytes=1 << 30, max_len=1 << 20), L.ERR_ARG), (dict(packed_proj=P + 8), L.ERR_ARG),
    (dict(packed_qkv=P + 4), L.ERR_ARG), (dict(input=P + 4), L.ERR_UNSUPPORTED), (dict(input_stride=258), L.ERR_UNSUPPORTED),
    (dict(combined_work=P + 4), L.ERR_ARG), (dict(batch=65535, max_new=1 << 20), L.ERR_LIMIT)])
def test_a_step_that_is_refused_has_launched_nothing(bad, want):
    """The later parts' refusals too come before the first launch (which fails here, for want of a GPU, as ERR_CUDA)."""
    assert L.load().fblt_paged_self_attention_step(C.byref(step(**bad)), None) == want


def test_a_split_call_wants_an_aligned_workspace():
    d = attn(max_len=1 << 20)
    assert L.load().fblt_paged_attn_workspace(C.byref(d)) > 0  # the plan splits
    assert L.load().fblt_paged_attn(C.byref(d), P + 8, 1 << 30, None) == L.ERR_ARG
    assert L.load().fblt_paged_attn(C.byref(d), P, 16, None) == L.ERR_WORKSPACE
