"""Host-side mirror of the reference's attention operator interface over the C ABI.

Names follow the reference: `attention_head_core` is blt_attention_head_core
(ops/attn_core.h:46) on the CUDA backend; `MaskConfig` is the batched
blt_mask_config (ops/mask_builder.h:12-32); `attn_forward` / `attn_decode`
replace the per-head loops of models/attention.c:199-202,
models/cross_attention.c:147-150 and infer/kv_cache.c:303-324,369-390.

torch is used only to own device memory and streams; every computation goes
through libfblt_attn.so.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import lib as L


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    if isinstance(t, torch.Tensor):
        return t.data_ptr()
    if isinstance(t, np.ndarray):
        return t.ctypes.data
    raise TypeError(type(t))


# the current stream's handle without an object around it (a microsecond of a decode step's call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        return _raw_stream(torch.cuda.current_device()) or None
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream or None
    return stream


# --------------------------------------------------------------------------- L0

def attention_head_core(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, combined: torch.Tensor, *,
                        col_offset: int, head_dim: int, scale: float, is_causal: bool = False,
                        mask: Optional[torch.Tensor] = None, weights_out: Optional[torch.Tensor] = None,
                        lse_out: Optional[torch.Tensor] = None, scores_scratch: Optional[torch.Tensor] = None,
                        fatal: bool = False) -> None:
    """One head of one sequence. q/k/v are 2-D fp32 CUDA views whose first column is the
    head's first column (row stride = .stride(0)); `combined` is the full [nq, E] output
    buffer and only `head_dim` columns at `col_offset` are written.

    fatal=True goes through the reference-named symbol (errors exit the process, as in
    the reference); otherwise the status-returning twin is used.
    """
    lib = L.load()
    a = L.HeadArgs()
    a.q, a.q_stride = q.data_ptr(), q.stride(0)
    a.k, a.k_stride = k.data_ptr(), k.stride(0)
    a.v, a.v_stride = v.data_ptr(), v.stride(0)
    a.combined, a.combined_stride, a.combined_col_offset = combined.data_ptr(), combined.stride(0), col_offset
    a.weights_out = _ptr(weights_out)
    a.lse_out = _ptr(lse_out)
    a.scores_scratch = _ptr(scores_scratch)
    a.mask = _ptr(mask)
    a.nq, a.nk, a.head_dim = q.shape[0], k.shape[0], head_dim
    a.is_causal, a.scale = bool(is_causal), float(scale)
    if fatal:
        lib.blt_attention_head_core_cuda(L.BACKEND_CUDA, C.byref(a))
    else:
        L.check(lib.fblt_attention_head(C.byref(a), _stream_ptr(None)))


# --------------------------------------------------------------------------- patches

def patch_bounds(starts: Sequence[int], lengths: Sequence[int], seq_len: int) -> np.ndarray:
    """Boundary array [P+1] from (start_idx, length) pairs, validated like the reference
    validates tiling (ops/patch_pool_cpu.c:98-112)."""
    lib = L.load()
    n = len(starts)
    arr = (L.PatchInfo * max(n, 1))()
    for i, (s, ln) in enumerate(zip(starts, lengths)):
        arr[i].start_idx, arr[i].length, arr[i].peak_entropy = int(s), int(ln), 0.0
    out = np.zeros(n + 1, dtype=np.int32)
    L.check(lib.fblt_patch_bounds(arr, n, seq_len, out.ctypes.data_as(L.c_i32_p)))
    return out


def patch_latent_at(bounds: np.ndarray, pos: int) -> int:
    b = np.ascontiguousarray(bounds, dtype=np.int32)
    return int(L.load().fblt_patch_latent_at(b.ctypes.data_as(L.c_i32_p), len(b) - 1, int(pos)))


# --------------------------------------------------------------------------- masks

@dataclass
class MaskConfig:
    """Batched blt_mask_config. Per-sequence lists hold one numpy array per sequence."""
    is_causal: bool = False
    sliding_window: int = 0
    group_rule: int = L.GROUP_NONE
    subtokens: int = 1
    bidirectional_within_group: bool = True
    causal_offset: Optional[Sequence[int]] = None          # [batch]
    doc_bounds: Optional[List[np.ndarray]] = None           # per sequence: first position of doc d+1
    patch_bounds: Optional[List[np.ndarray]] = None         # per sequence: [P+1]
    q_pos_offset: Optional[Sequence[int]] = None            # [batch]
    trailing_closed: Optional[Sequence[int]] = None         # [batch]
    num_clean: Optional[Sequence[int]] = None               # [batch] -> block-diffusion INFER rule
    q_group_ids: Optional[np.ndarray] = None                # [total q rows]
    k_group_ids: Optional[np.ndarray] = None                # [total k rows]

    def host_tables(self, batch: int):
        """int32 numpy tables in the layout the C descriptor wants."""
        t = {}

        def i32(x):
            return np.ascontiguousarray(np.asarray(x, dtype=np.int32))

        if self.causal_offset is not None:
            t["causal_offset"] = i32(self.causal_offset)
        if self.doc_bounds is not None:
            cu = np.zeros(batch + 1, dtype=np.int32)
            cu[1:] = np.cumsum([len(d) for d in self.doc_bounds])
            flat = np.concatenate([i32(d) for d in self.doc_bounds]) if cu[-1] else np.zeros(1, np.int32)
            t["cu_doc"], t["doc_bounds"] = cu, i32(flat)
        if self.patch_bounds is not None:
            cu = np.zeros(batch + 1, dtype=np.int32)
            cu[1:] = np.cumsum([len(p) for p in self.patch_bounds])
            t["cu_patch"], t["patch_bounds"] = cu, i32(np.concatenate([i32(p) for p in self.patch_bounds]))
        if self.q_pos_offset is not None:
            t["q_pos_offset"] = i32(self.q_pos_offset)
        if self.trailing_closed is not None:
            t["trailing_closed"] = np.ascontiguousarray(np.asarray(self.trailing_closed, dtype=np.uint8))
        if self.num_clean is not None:
            t["num_clean"] = i32(self.num_clean)
        if self.q_group_ids is not None:
            t["q_group_ids"] = i32(self.q_group_ids)
        if self.k_group_ids is not None:
            t["k_group_ids"] = i32(self.k_group_ids)
        return t

    def fill(self, m: L.MaskDesc, tables: dict) -> None:
        m.is_causal = int(self.is_causal)
        m.sliding_window = int(self.sliding_window)
        m.group_rule = int(self.group_rule)
        m.subtokens = int(self.subtokens)
        m.bidirectional_within_group = int(self.bidirectional_within_group)
        for name in ("causal_offset", "cu_doc", "doc_bounds", "cu_patch", "patch_bounds", "q_pos_offset",
                     "trailing_closed", "q_group_ids", "k_group_ids", "num_clean"):
            setattr(m, name, _ptr(tables.get(name)))


@dataclass
class AttnBatch:
    """Device-resident descriptor of one batched forward call; keeps its tables alive."""
    desc: L.AttnDesc
    keep: list = field(default_factory=list)


def make_batch(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, cu_q: Sequence[int],
               cu_k: Sequence[int], num_heads: int, head_dim: int, scale: float,
               mask: Optional[MaskConfig] = None, impl: int = L.IMPL_AUTO, precision: int = L.PREC_FP32,
               rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
               rope_q_pos: Optional[torch.Tensor] = None, rope_k_pos: Optional[torch.Tensor] = None) -> AttnBatch:
    """q/k/v/out: 2-D fp32 CUDA views (rows packed over sequences, row stride = .stride(0),
    first column = head 0). cu_q / cu_k: row offsets [batch+1] (host)."""
    dev = q.device
    cu_q_h = np.asarray(cu_q, dtype=np.int32)
    cu_k_h = np.asarray(cu_k, dtype=np.int32)
    batch = len(cu_q_h) - 1
    mask = mask or MaskConfig()
    d = L.AttnDesc()
    d.batch, d.num_heads, d.head_dim = batch, num_heads, head_dim
    d.max_q = int(np.max(np.diff(cu_q_h))) if batch else 0
    d.max_k = int(np.max(np.diff(cu_k_h))) if batch else 0
    d.impl, d.precision = impl, precision
    d.total_q_rows = int(cu_q_h[-1]) if batch else 0       # where the tensors end: the TMA-loading kernel needs it
    d.total_k_rows = int(cu_k_h[-1]) if batch else 0
    keep = []

    def dev_i32(a):
        t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        keep.append(t)
        return t

    d.cu_q = dev_i32(cu_q_h).data_ptr()
    d.cu_k = dev_i32(cu_k_h).data_ptr()
    d.q, d.q_stride = q.data_ptr(), q.stride(0)
    d.k, d.k_stride = k.data_ptr(), k.stride(0)
    d.v, d.v_stride = v.data_ptr(), v.stride(0)
    d.out, d.out_stride = out.data_ptr(), out.stride(0)
    d.scale = float(scale)
    tables = {name: dev_i32(arr) for name, arr in mask.host_tables(batch).items()}
    mask.fill(d.mask, tables)
    if rope_cos is not None:
        d.rope_cos, d.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
        keep += [rope_cos, rope_sin]
        if rope_q_pos is not None:
            d.rope_q_pos = rope_q_pos.data_ptr()
            keep.append(rope_q_pos)
        if rope_k_pos is not None:
            d.rope_k_pos = rope_k_pos.data_ptr()
            keep.append(rope_k_pos)
    keep += [q, k, v, out]
    return AttnBatch(d, keep)


def attn_forward(batch: AttnBatch, stream=None) -> None:
    L.check(L.load().fblt_attn_forward(C.byref(batch.desc), _stream_ptr(stream)))


def mask_bitmap(batch: AttnBatch, use_range: bool = False) -> torch.Tensor:
    """uint8 [batch, max_q, max_k] of allowed(i, j), evaluated by the library on the device."""
    d = batch.desc
    bm = torch.zeros((d.batch, d.max_q, d.max_k), dtype=torch.uint8, device="cuda")
    L.check(L.load().fblt_mask_bitmap(C.byref(d), bm.data_ptr(), int(use_range), _stream_ptr(None)))
    return bm


def mask_materialize(batch: AttnBatch, seq: int):
    d = batch.desc
    cu_q = batch.keep[0].cpu().numpy()
    cu_k = batch.keep[1].cpu().numpy()
    nq, nk = int(cu_q[seq + 1] - cu_q[seq]), int(cu_k[seq + 1] - cu_k[seq])
    m = torch.empty((nq, nk), dtype=torch.float32, device="cuda")
    empty = C.c_int32(0)
    L.check(L.load().fblt_mask_materialize(C.byref(d), seq, m.data_ptr(), C.byref(empty), _stream_ptr(None)))
    return m, empty.value


def _host_sizes(a):
    """Host size_t array (the reference passes its id arrays as host pointers) or None."""
    if a is None:
        return None
    return np.ascontiguousarray(np.asarray(a, dtype=np.uint64))


def build_attention_mask(nq: int, nk: int, *, window: int = 0, doc_boundaries=None, q_groups=None, k_groups=None,
                         bidirectional: bool = True, is_causal: bool = False, causal_offset: int = 0, stream=None):
    """blt_build_attention_mask on the CUDA backend: dense [nq, nk] 0 / -inf tensor and the number of
    query rows without an allowed key (fatal in the reference, ops/mask_builder_cpu.c:93)."""
    lib = L.load()
    c = L.MaskConfig()
    c.seq_len_q, c.seq_len_kv, c.sliding_window = nq, nk, window
    db, qg, kg = _host_sizes(doc_boundaries), _host_sizes(q_groups), _host_sizes(k_groups)
    if db is not None:
        c.doc_boundaries, c.num_docs = db.ctypes.data, len(db) + 1
    if qg is not None:
        c.query_group_ids, c.kv_group_ids = qg.ctypes.data, kg.ctypes.data
    c.bidirectional_within_group, c.is_causal, c.causal_offset = bool(bidirectional), bool(is_causal), causal_offset
    need = lib.fblt_mask_dense_scratch_bytes(C.byref(c))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    m = torch.full((nq, nk), float("nan"), dtype=torch.float32, device="cuda")
    empty = C.c_int32(-1)
    L.check(lib.fblt_build_attention_mask_dense(C.byref(c), m.data_ptr(), scratch.data_ptr(), need, C.byref(empty),
                                                _stream_ptr(stream)))
    return m, empty.value


def build_block_diffusion_mask(mode: int, S: int, N: int, B: int = 0, block_starts=None, stream=None):
    """blt_build_block_diffusion_mask on the CUDA backend (mode 0 = TRAIN, 1 = INFER): [S, S] and the
    number of empty rows."""
    lib = L.load()
    c = L.BlockDiffusionConfig()
    c.mode, c.seq_len, c.num_clean, c.block_size = mode, S, N, B
    bs = _host_sizes(block_starts)
    if bs is not None:
        c.block_starts, c.num_blocks = bs.ctypes.data, len(bs)
    need = lib.fblt_block_diffusion_mask_scratch_bytes(C.byref(c))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    m = torch.full((S, S), float("nan"), dtype=torch.float32, device="cuda")
    empty = C.c_int32(-1)
    L.check(lib.fblt_build_block_diffusion_mask_dense(C.byref(c), m.data_ptr(), scratch.data_ptr(), need,
                                                      C.byref(empty), _stream_ptr(stream)))
    return m, empty.value


# --------------------------------------------------------------------------- decode

def make_decode(k_cache: torch.Tensor, v_cache: torch.Tensor, base_len: torch.Tensor, q: torch.Tensor,
                out: torch.Tensor, num_heads: int, head_dim: int, n_new: int, scale: float, *,
                block_mode: bool = False, window: int = 0, k_new: Optional[torch.Tensor] = None,
                v_new: Optional[torch.Tensor] = None, max_len: Optional[int] = None, splits: int = 0,
                rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None) -> L.DecodeDesc:
    """k_cache / v_cache: [batch, cache_rows, E] fp32 CUDA; base_len: int32 CUDA [batch];
    q/out (and k_new/v_new): [batch * n_new, E]."""
    d = L.DecodeDesc()
    d.batch, d.num_heads, d.head_dim, d.n_new = k_cache.shape[0], num_heads, head_dim, n_new
    d.block_mode, d.window = int(block_mode), int(window)
    d.max_len = int(max_len) if max_len is not None else int(k_cache.shape[1])
    d.splits = splits
    d.base_len = base_len.data_ptr()
    d.k_cache, d.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    d.cache_seq_stride, d.cache_row_stride = k_cache.stride(0), k_cache.stride(1)
    d.q, d.q_stride = q.data_ptr(), q.stride(0)
    if k_new is not None:
        d.k_new, d.v_new, d.kv_new_stride = k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0)
    d.out, d.out_stride = out.data_ptr(), out.stride(0)
    d.scale = float(scale)
    if rope_cos is not None:
        d.rope_cos, d.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    return d


def decode_workspace(d: L.DecodeDesc) -> Optional[torch.Tensor]:
    n = L.load().fblt_attn_decode_workspace(C.byref(d))
    return torch.empty(n, dtype=torch.uint8, device="cuda") if n else None


def attn_decode(d: L.DecodeDesc, workspace: Optional[torch.Tensor] = None, stream=None) -> None:
    wp = workspace.data_ptr() if workspace is not None else None
    wn = workspace.numel() if workspace is not None else 0
    L.check(L.load().fblt_attn_decode(C.byref(d), wp, wn, _stream_ptr(stream)))


# --------------------------------------------------------------------------- decisions

def argmax_rows(logits: torch.Tensor) -> torch.Tensor:
    ids = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    L.check(L.load().fblt_argmax_rows(logits.data_ptr(), logits.stride(0), logits.shape[0], logits.shape[1],
                                      ids.data_ptr(), _stream_ptr(None)))
    return ids


class PackedWeights:
    """b [K, N] packed for fblt_matmul (device buffer + shape)."""

    def __init__(self, b: torch.Tensor):
        assert b.dim() == 2 and b.dtype == torch.float32 and b.is_cuda and b.stride(1) == 1
        self.K, self.N = int(b.shape[0]), int(b.shape[1])
        lib = L.load()
        nbytes = lib.fblt_matmul_packed_bytes(self.K, self.N)
        self.buf = torch.empty(nbytes, dtype=torch.uint8, device=b.device)
        L.check(lib.fblt_matmul_pack_weights(b.data_ptr(), b.stride(0), self.K, self.N, self.buf.data_ptr(), nbytes,
                                             _stream_ptr(None)))


def matmul(a: torch.Tensor, w: PackedWeights, out: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
           precision: int = L.PREC_FP32) -> torch.Tensor:
    """out = a @ b (+ bias) with b given as PackedWeights; a [M, K] float32 with unit column stride."""
    assert a.dim() == 2 and a.dtype == torch.float32 and a.stride(1) == 1 and a.shape[1] == w.K
    if out is None:
        out = torch.empty(a.shape[0], w.N, dtype=torch.float32, device=a.device)
    L.check(L.load().fblt_matmul(a.data_ptr(), a.stride(0), w.buf.data_ptr(), bias.data_ptr() if bias is not None else None,
                                 out.data_ptr(), out.stride(0), a.shape[0], w.K, w.N, precision, _stream_ptr(None)))
    return out


def mha_forward(x: torch.Tensor, w_qkv: PackedWeights, w_proj: PackedWeights, cu_rows: Sequence[int], num_heads: int,
                mask: Optional[MaskConfig] = None, rope_cos: Optional[torch.Tensor] = None,
                rope_sin: Optional[torch.Tensor] = None, precision: int = L.PREC_FP32) -> torch.Tensor:
    """The multi-head self-attention block over packed sequences (x [rows, E]); returns [rows, E]."""
    rows, E = int(x.shape[0]), int(x.shape[1])
    dev = x.device
    cu_h = np.asarray(cu_rows, dtype=np.int32)
    batch = len(cu_h) - 1
    mask = mask or MaskConfig()
    d = L.MhaDesc()
    d.batch, d.num_heads, d.head_dim = batch, num_heads, E // num_heads
    d.max_len = int(np.max(np.diff(cu_h))) if batch else 0
    d.total_rows = rows
    keep = []

    def dev_i32(a):
        t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        keep.append(t)
        return t

    d.cu_rows = dev_i32(cu_h).data_ptr()
    out = torch.empty(rows, E, dtype=torch.float32, device=dev)
    qkv = torch.empty(rows, 3 * E, dtype=torch.float32, device=dev)
    comb = torch.empty(rows, E, dtype=torch.float32, device=dev)
    d.input, d.input_stride = x.data_ptr(), x.stride(0)
    d.packed_qkv, d.packed_proj = w_qkv.buf.data_ptr(), w_proj.buf.data_ptr()
    d.output, d.output_stride = out.data_ptr(), out.stride(0)
    d.qkv_work, d.combined_work = qkv.data_ptr(), comb.data_ptr()
    tables = {name: dev_i32(arr) for name, arr in mask.host_tables(batch).items()}
    mask.fill(d.mask, tables)
    if rope_cos is not None:
        d.rope_cos, d.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    d.precision = precision
    L.check(L.load().fblt_mha_forward(C.byref(d), _stream_ptr(None)))
    torch.cuda.current_stream().synchronize()   # the scratch tensors above die with this call
    return out


def cross_attention_forward(query_in: torch.Tensor, kv_in: torch.Tensor, w_q: PackedWeights, w_kv: PackedWeights,
                            w_proj: PackedWeights, cu_q: Sequence[int], cu_k: Sequence[int], num_heads: int,
                            mask: MaskConfig, precision: int = L.PREC_FP32) -> torch.Tensor:
    """The cross-attention block over packed sequences; w_kv packs [weight_k | weight_v] ([E, 2E])."""
    E = int(query_in.shape[1])
    dev = query_in.device
    cu_q_h, cu_k_h = np.asarray(cu_q, dtype=np.int32), np.asarray(cu_k, dtype=np.int32)
    batch = len(cu_q_h) - 1
    d = L.CrossDesc()
    d.batch, d.num_heads, d.head_dim = batch, num_heads, E // num_heads
    d.max_q = int(np.max(np.diff(cu_q_h))) if batch else 0
    d.max_k = int(np.max(np.diff(cu_k_h))) if batch else 0
    d.precision = precision
    d.total_q_rows, d.total_k_rows = int(query_in.shape[0]), int(kv_in.shape[0])
    keep = []

    def dev_i32(a):
        t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        keep.append(t)
        return t

    d.cu_q, d.cu_k = dev_i32(cu_q_h).data_ptr(), dev_i32(cu_k_h).data_ptr()
    out = torch.empty(d.total_q_rows, E, dtype=torch.float32, device=dev)
    qw = torch.empty(d.total_q_rows, E, dtype=torch.float32, device=dev)
    kvw = torch.empty(d.total_k_rows, 2 * E, dtype=torch.float32, device=dev)
    comb = torch.empty(d.total_q_rows, E, dtype=torch.float32, device=dev)
    d.query_in, d.query_stride = query_in.data_ptr(), query_in.stride(0)
    d.kv_in, d.kv_stride = kv_in.data_ptr(), kv_in.stride(0)
    d.packed_q, d.packed_kv, d.packed_proj = w_q.buf.data_ptr(), w_kv.buf.data_ptr(), w_proj.buf.data_ptr()
    d.output, d.output_stride = out.data_ptr(), out.stride(0)
    d.q_work, d.kv_work, d.combined_work = qw.data_ptr(), kvw.data_ptr(), comb.data_ptr()
    tables = {name: dev_i32(arr) for name, arr in mask.host_tables(batch).items()}
    mask.fill(d.mask, tables)
    L.check(L.load().fblt_cross_attention_forward(C.byref(d), _stream_ptr(None)))
    torch.cuda.current_stream().synchronize()   # the scratch tensors above die with this call
    return out


def kv_self_attention_step(x: torch.Tensor, w_qkv: PackedWeights, w_proj: PackedWeights, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, base_len: torch.Tensor, num_heads: int, n_new: int, *,
                           rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                           block_mode: bool = False, window: int = 0, max_len: int = 0,
                           precision: int = L.PREC_FP32) -> torch.Tensor:
    """Self-attention part of a decode step: x [batch*n_new, E] rows -> [batch*n_new, E]; K/V rows are
    written into the caches ([batch, rows, E]) at base_len .. base_len + n_new."""
    rows, E = int(x.shape[0]), int(x.shape[1])
    dev = x.device
    d = L.KvStepDesc()
    d.batch, d.num_heads, d.head_dim, d.n_new = rows // n_new, num_heads, E // num_heads, n_new
    d.block_mode, d.window, d.precision = int(block_mode), window, precision
    d.max_len = max_len or int(k_cache.shape[1])
    d.base_len = base_len.data_ptr()
    d.k_cache, d.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    d.cache_seq_stride, d.cache_row_stride = k_cache.stride(0), k_cache.stride(1)
    out = torch.empty(rows, E, dtype=torch.float32, device=dev)
    qkv = torch.empty(rows, 3 * E, dtype=torch.float32, device=dev)
    comb = torch.empty(rows, E, dtype=torch.float32, device=dev)
    ws = torch.empty(8 << 20, dtype=torch.uint8, device=dev)
    d.input, d.input_stride = x.data_ptr(), x.stride(0)
    d.packed_qkv, d.packed_proj = w_qkv.buf.data_ptr(), w_proj.buf.data_ptr()
    d.output, d.output_stride = out.data_ptr(), out.stride(0)
    d.qkv_work, d.combined_work = qkv.data_ptr(), comb.data_ptr()
    d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
    if rope_cos is not None:
        d.rope_cos, d.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()
    L.check(L.load().fblt_kv_self_attention_step(C.byref(d), _stream_ptr(None)))
    torch.cuda.current_stream().synchronize()   # the scratch tensors above die with this call
    return out


class KvStepPlan:
    """The decode-step block with every buffer allocated up front: run() only enqueues the three
    launches (no allocation, no synchronisation), so a loop of steps can be captured once in a CUDA
    graph and replayed while the caches grow -- the cache lengths are read from device memory
    (base_len), not baked into the launches. x is the static input [batch*n_new, E]; out the static
    output. max_len must bound base_len + n_new over every replay (default: the cache capacity)."""

    def __init__(self, w_qkv: PackedWeights, w_proj: PackedWeights, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 base_len: torch.Tensor, num_heads: int, n_new: int, *, rope_cos: Optional[torch.Tensor] = None,
                 rope_sin: Optional[torch.Tensor] = None, block_mode: bool = False, window: int = 0,
                 max_len: int = 0, precision: int = L.PREC_FP32):
        batch, E, dev = int(k_cache.shape[0]), int(k_cache.shape[2]), k_cache.device
        rows = batch * n_new
        self.x = torch.zeros(rows, E, dtype=torch.float32, device=dev)
        self.out = torch.empty(rows, E, dtype=torch.float32, device=dev)
        self._qkv = torch.empty(rows, 3 * E, dtype=torch.float32, device=dev)
        self._comb = torch.empty(rows, E, dtype=torch.float32, device=dev)
        self._ws = torch.empty(8 << 20, dtype=torch.uint8, device=dev)
        self._keep = [w_qkv, w_proj, k_cache, v_cache, base_len, rope_cos, rope_sin]
        d = self.desc = L.KvStepDesc()
        d.batch, d.num_heads, d.head_dim, d.n_new = batch, num_heads, E // num_heads, n_new
        d.block_mode, d.window, d.precision = int(block_mode), window, precision
        d.max_len = max_len or int(k_cache.shape[1])
        d.base_len = base_len.data_ptr()
        d.k_cache, d.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        d.cache_seq_stride, d.cache_row_stride = k_cache.stride(0), k_cache.stride(1)
        d.input, d.input_stride = self.x.data_ptr(), self.x.stride(0)
        d.packed_qkv, d.packed_proj = w_qkv.buf.data_ptr(), w_proj.buf.data_ptr()
        d.output, d.output_stride = self.out.data_ptr(), self.out.stride(0)
        d.qkv_work, d.combined_work = self._qkv.data_ptr(), self._comb.data_ptr()
        d.workspace, d.workspace_bytes = self._ws.data_ptr(), self._ws.numel()
        if rope_cos is not None:
            d.rope_cos, d.rope_sin = rope_cos.data_ptr(), rope_sin.data_ptr()

    def run(self, stream=None) -> None:
        L.check(L.load().fblt_kv_self_attention_step(C.byref(self.desc), _stream_ptr(stream)))


def unmask_step(logits: torch.Tensor, masked: torch.Tensor, tokens: torch.Tensor, strategy: int, threshold: float):
    """One unmask round over a batch of candidates. logits [batch*B, V] float32, masked/tokens
    [batch, B] uint8 (updated in place). Returns (sel [batch] int64 bit masks, conf [batch,B],
    ent [batch,B], remaining [batch])."""
    batch, B = masked.shape
    dev = logits.device
    sel = torch.empty(batch, dtype=torch.int32, device=dev)          # same bits as the uint32 the kernel writes
    conf = torch.empty(batch, B, dtype=torch.float32, device=dev)
    ent = torch.empty(batch, B, dtype=torch.float32, device=dev)
    left = torch.empty(batch, dtype=torch.int32, device=dev)
    L.check(L.load().fblt_unmask_step(logits.data_ptr(), logits.stride(0), batch, B, logits.shape[1], strategy,
                                      float(threshold), masked.data_ptr(), tokens.data_ptr(), sel.data_ptr(),
                                      conf.data_ptr(), ent.data_ptr(), left.data_ptr(), _stream_ptr(None)))
    return sel.to(torch.int64) & 0xFFFFFFFF, conf, ent, left


def verify_accept(x: torch.Tensor, pred: torch.Tensor, l: torch.Tensor, r: torch.Tensor, target_len: torch.Tensor):
    """In-place accept-until-mismatch over a batch of candidates; returns (new_len, accepted)."""
    batch = x.shape[0]
    new_len = torch.empty(batch, dtype=torch.int32, device=x.device)
    accepted = torch.empty(batch, dtype=torch.int32, device=x.device)
    L.check(L.load().fblt_verify_accept(x.data_ptr(), x.stride(0), pred.data_ptr(), pred.stride(0), l.data_ptr(),
                                        r.data_ptr(), target_len.data_ptr(), batch, new_len.data_ptr(),
                                        accepted.data_ptr(), _stream_ptr(None)))
    return new_len, accepted


def dv_commit(logits: torch.Tensor, width: int, x: torch.Tensor, l: torch.Tensor, r: torch.Tensor,
              target_len: torch.Tensor, cache_len: torch.Tensor, stream=None) -> torch.Tensor:
    """One batched verify-and-commit round on the device (fblt_dv_commit): x, l and cache_len are
    updated in place; returns the accepted counts. logits: [batch * width, vocab]."""
    batch = x.shape[0]
    accepted = torch.empty(batch, dtype=torch.int32, device=x.device)
    pred = torch.empty(batch * width, dtype=torch.int32, device=x.device)
    L.check(L.load().fblt_dv_commit(logits.data_ptr(), logits.stride(0), width, logits.shape[1], batch, x.data_ptr(),
                                    x.stride(0), l.data_ptr(), r.data_ptr(), target_len.data_ptr(), cache_len.data_ptr(),
                                    accepted.data_ptr(), pred.data_ptr(), _stream_ptr(stream)))
    return accepted


# --------------------------------------------------------------------------- paged 8-bit KV cache
# The make_* functions check their tensors and fill a descriptor that keeps them alive (`keep`); it is made once for a
# program's buffers and launched as often as it likes.


def _keep(d, *tensors):
    """Keeps the tensors of a descriptor alive and notes the device that all of them have to be on."""
    d.keep = tensors
    devices = {t.device.index for t in tensors if isinstance(t, torch.Tensor)}
    devices |= {t.k_codes.device.index for t in tensors if isinstance(t, PagedKvCache)}
    if len(devices) != 1:
        raise ValueError(f"tensors on different devices: {sorted(devices)}")
    d.device = devices.pop()
    return d


def _stream_on(d, stream) -> Optional[int]:
    """The stream's handle; kernels are launched on the current device, where the descriptor's tensors have to be."""
    current = torch.cuda.current_device()
    if current != d.device or (isinstance(stream, torch.cuda.Stream) and stream.device_index != current):
        raise ValueError(f"tensors on device {d.device}, current device {current}, stream {stream}")
    return _raw_stream(current) or None if stream is None else _stream_ptr(stream)


_KV_FORMATS = {"e4m3": L.KV_E4M3, "int8": L.KV_INT8}


def _rows(t: torch.Tensor, cols: int, what: str, dtypes=(torch.float32,)) -> torch.Tensor:
    """Checks a 2-D row view that is handed to the library by pointer and row stride."""
    if not (t.is_cuda and t.dim() == 2 and t.dtype in dtypes and t.shape[1] == cols and (t.stride(1) == 1 or cols == 1)):
        raise ValueError(f"{what}: a CUDA [rows, {cols}] view of {'/'.join(str(d) for d in dtypes)} with unit column stride is needed")
    return t


def _row_stride(t: torch.Tensor) -> int:
    """Row stride of a view that _rows has passed; a single row's is any number at all (a transposed column's is 1)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _table(t: torch.Tensor, n: int, what: str) -> torch.Tensor:
    if not (t.is_cuda and t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] >= n and (t.stride(0) == 1 or n <= 1)):
        raise ValueError(f"{what}: a contiguous CUDA int32 tensor of {n} entries is needed")
    return t


def _vector(t: Optional[torch.Tensor], n: int, what: str) -> Optional[int]:
    if t is None:
        return None
    if not (t.is_cuda and t.dtype == torch.float32 and t.shape == (n,) and t.is_contiguous()):
        raise ValueError(f"{what}: a contiguous CUDA float32 tensor of {n} values is needed")
    return t.data_ptr()


def _rope(d, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], head_dim: int) -> None:
    if (cos is None) != (sin is None):
        raise ValueError("rope_cos and rope_sin go together")
    if cos is None:
        return
    for t in (cos, sin):
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and t.dim() == 2
                and t.shape[1] == head_dim // 2 and t.shape[0] == cos.shape[0]):
            raise ValueError(f"rotary tables: contiguous CUDA float32 [positions, {head_dim // 2}] tensors are needed")
    d.rope_cos, d.rope_sin, d.rope_len = cos.data_ptr(), sin.data_ptr(), int(cos.shape[0])


class PagedKvCache:
    """K and V in 8 bits with one power-of-two exponent for every (position, kv head), in pages.

    k_codes / v_codes: uint8 [num_pages, num_kv_heads, page_size, head_dim]; k_exp / v_exp: int8 [num_pages,
    num_kv_heads, page_size]; page_table: int32 [batch, max_pages], page of positions j * page_size ... of a sequence (rows of
    their own: sequences share pages, not table rows). All on one device.
    fmt: "e4m3" or "int8". `status` collects the FBLT_PAGED_* bits that kernels raise (status_bits() reads them)."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_exp: torch.Tensor, v_exp: torch.Tensor,
                 page_table: torch.Tensor, fmt: str):
        if fmt not in _KV_FORMATS:
            raise ValueError(f"fmt {fmt!r} (e4m3 or int8)")
        shape = k_codes.shape
        if k_codes.dim() != 4 or v_codes.shape != shape or k_exp.shape != shape[:3] or v_exp.shape != shape[:3]:
            raise ValueError("codes are [pages, kv_heads, page_size, head_dim], exponents [pages, kv_heads, page_size]")
        for t, dt in ((k_codes, torch.uint8), (v_codes, torch.uint8), (k_exp, torch.int8), (v_exp, torch.int8)):
            if not (t.is_cuda and t.dtype == dt and t.is_contiguous()):
                raise ValueError("codes are contiguous CUDA uint8 tensors, exponents int8")
        if not (page_table.is_cuda and page_table.dtype == torch.int32 and page_table.dim() == 2
                and (page_table.stride(1) == 1 or page_table.shape[1] == 1)):
            raise ValueError("page_table: a CUDA int32 [batch, max_pages] tensor with unit column stride is needed")
        if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("page_table: rows that overlap (an expanded table); every sequence needs a row of its own")
        if len({t.device for t in (k_codes, v_codes, k_exp, v_exp, page_table)}) != 1:
            raise ValueError("codes, exponents and page_table: tensors on different devices")
        self.k_codes, self.v_codes, self.k_exp, self.v_exp, self.page_table, self.fmt = k_codes, v_codes, k_exp, v_exp, page_table, fmt
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = (int(n) for n in shape)
        self.batch = int(page_table.shape[0])
        self.status = torch.zeros(1, dtype=torch.int32, device=k_codes.device)
        c = self.desc = L.PagedCache()
        c.format, c.num_kv_heads, c.head_dim, c.page_size = _KV_FORMATS[fmt], self.num_kv_heads, self.head_dim, self.page_size
        c.num_pages, c.max_pages = self.num_pages, int(page_table.shape[1])
        c.k_codes, c.v_codes, c.k_exp, c.v_exp = k_codes.data_ptr(), v_codes.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr()
        c.page_table, c.page_table_stride = page_table.data_ptr(), max(page_table.stride(0), int(page_table.shape[1]))
        c.status = self.status.data_ptr()

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, page_table: torch.Tensor, fmt: str) -> "PagedKvCache":
        """A pool of zeroed pages on the page table's device."""
        dev = page_table.device
        codes = [torch.zeros(num_pages, num_kv_heads, page_size, head_dim, dtype=torch.uint8, device=dev) for _ in range(2)]
        exps = [torch.zeros(num_pages, num_kv_heads, page_size, dtype=torch.int8, device=dev) for _ in range(2)]
        return cls(*codes, *exps, page_table, fmt)

    def status_bits(self) -> int:
        """The status word (waits for the device); it is cleared."""
        bits = int(self.status.item())
        self.status.zero_()
        return bits


def make_qk_norm_rope(q: Optional[torch.Tensor], k: Optional[torch.Tensor], pos: Optional[torch.Tensor], num_heads: int,
                      num_kv_heads: int, head_dim: int, *, q_out: Optional[torch.Tensor] = None,
                      k_out: Optional[torch.Tensor] = None, q_gain: Optional[torch.Tensor] = None,
                      k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6, rope_cos: Optional[torch.Tensor] = None,
                      rope_sin: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> L.QkNormRopeDesc:
    """q [rows, num_heads * head_dim] and k [rows, num_kv_heads * head_dim] (views of a packed projection will do);
    without q_out / k_out the rows are changed in place. pos: int32 [rows]."""
    d = L.QkNormRopeDesc()
    rows = int((q if q is not None else k).shape[0])
    d.rows, d.num_heads, d.num_kv_heads, d.head_dim, d.eps = rows, num_heads, num_kv_heads, head_dim, float(eps)
    for name, x, out, heads in (("q", q, q_out, num_heads), ("k", k, k_out, num_kv_heads)):
        if x is None:
            continue
        out = x if out is None else out
        for t in (_rows(x, heads * head_dim, name), _rows(out, heads * head_dim, name + "_out")):
            if t.shape[0] != rows:
                raise ValueError("q, k and their outputs have one row count")
        setattr(d, name, x.data_ptr())
        setattr(d, name + "_stride", _row_stride(x))
        setattr(d, name + "_out", out.data_ptr())
        setattr(d, name + "_out_stride", _row_stride(out))
    d.q_gain, d.k_gain = _vector(q_gain, head_dim, "q_gain"), _vector(k_gain, head_dim, "k_gain")
    _rope(d, rope_cos, rope_sin, head_dim)
    if pos is not None:
        d.pos = _table(pos, rows, "pos").data_ptr()
    if status is not None:
        d.status = _table(status, 1, "status").data_ptr()
    return _keep(d, q, k, pos, q_out, k_out, q_gain, k_gain, rope_cos, rope_sin, status)


def qk_norm_rope(d: L.QkNormRopeDesc, stream=None) -> None:
    L.check(L.load().fblt_qk_norm_rope(C.byref(d), _stream_on(d, stream)))


def make_paged_append(cache: PagedKvCache, cu_new: torch.Tensor, base_len: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                      q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, num_heads: int = 0,
                      q_gain: Optional[torch.Tensor] = None, k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None) -> L.PagedAppendDesc:
    """k / v: [rows, kv_heads * head_dim], packed by sequence (cu_new int32 [batch + 1]) at positions base_len[b] + i.
    With q ([rows, num_heads * head_dim]) the query rows are normalised and rotated too (into q_out, or in place)."""
    d = L.PagedAppendDesc()
    hd, kc, rows = cache.head_dim, cache.num_kv_heads * cache.head_dim, int(k.shape[0])
    d.cache, d.batch, d.num_heads, d.total_rows, d.eps = cache.desc, cache.batch, num_heads, rows, float(eps)
    d.cu_new, d.base_len = _table(cu_new, cache.batch + 1, "cu_new").data_ptr(), _table(base_len, cache.batch, "base_len").data_ptr()
    d.k, d.k_stride = _rows(k, kc, "k").data_ptr(), _row_stride(k)
    d.v, d.v_stride = _rows(v, kc, "v").data_ptr(), _row_stride(v)
    out = q if q_out is None else q_out
    if q is not None:
        d.q, d.q_stride = _rows(q, num_heads * hd, "q").data_ptr(), _row_stride(q)
        d.q_out, d.q_out_stride = _rows(out, num_heads * hd, "q_out").data_ptr(), _row_stride(out)
    if any(t is not None and t.shape[0] != rows for t in (v, q, out)):
        raise ValueError("q, q_out, k and v have one row count")
    d.q_gain, d.k_gain = _vector(q_gain, hd, "q_gain"), _vector(k_gain, hd, "k_gain")
    _rope(d, rope_cos, rope_sin, hd)
    return _keep(d, cache, cu_new, base_len, k, v, q, q_out, q_gain, k_gain, rope_cos, rope_sin)


def paged_append(d: L.PagedAppendDesc, stream=None) -> None:
    L.check(L.load().fblt_paged_append(C.byref(d), _stream_on(d, stream)))


def make_paged_read(cache: PagedKvCache, cu_rows: torch.Tensor, k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor], *,
                    start: Optional[torch.Tensor] = None) -> L.PagedReadDesc:
    """Positions start[b] (0 without `start`) .. of every sequence into packed rows of float32 or bfloat16 (both exact)."""
    d = L.PagedReadDesc()
    first = k_out if k_out is not None else v_out
    if first is None or (k_out is not None and v_out is not None and (k_out.dtype != v_out.dtype or k_out.shape != v_out.shape)):
        raise ValueError("k_out / v_out: at least one, of one shape and type")
    d.cache, d.batch, d.total_rows = cache.desc, cache.batch, int(first.shape[0])
    d.out_type = L.PAGED_OUT_BF16 if first.dtype == torch.bfloat16 else L.PAGED_OUT_FP32
    d.cu_rows = _table(cu_rows, cache.batch + 1, "cu_rows").data_ptr()
    d.start = None if start is None else _table(start, cache.batch, "start").data_ptr()
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            setattr(d, name, _rows(t, cache.num_kv_heads * cache.head_dim, name, (torch.float32, torch.bfloat16)).data_ptr())
            setattr(d, name + "_stride", _row_stride(t))
    return _keep(d, cache, cu_rows, k_out, v_out, start)


def paged_read(d: L.PagedReadDesc, stream=None) -> None:
    L.check(L.load().fblt_paged_read(C.byref(d), _stream_on(d, stream)))


def make_paged_attn(cache: PagedKvCache, cu_new: torch.Tensor, base_len: torch.Tensor, q: torch.Tensor, out: torch.Tensor,
                    num_heads: int, max_new: int, max_len: int, scale: float, *, block_mode: bool = False, window: int = 0,
                    splits: int = 0) -> L.PagedAttnDesc:
    """q / out: [rows, num_heads * head_dim], packed by sequence; row cu_new[b] + i is at position base_len[b] + i and
    the cache holds the new rows already. max_new / max_len bound the new rows and base_len + new rows."""
    d = L.PagedAttnDesc()
    cols = num_heads * cache.head_dim
    d.cache, d.batch, d.num_heads, d.total_rows = cache.desc, cache.batch, num_heads, int(q.shape[0])
    d.max_new, d.max_len, d.block_mode, d.window, d.splits = max_new, max_len, int(block_mode), int(window), splits
    d.cu_new, d.base_len = _table(cu_new, cache.batch + 1, "cu_new").data_ptr(), _table(base_len, cache.batch, "base_len").data_ptr()
    d.q, d.q_stride = _rows(q, cols, "q").data_ptr(), _row_stride(q)
    d.out, d.out_stride = _rows(out, cols, "out").data_ptr(), _row_stride(out)
    if q.shape[0] != out.shape[0]:
        raise ValueError("q and out have one row count")
    d.scale = float(scale)
    return _keep(d, cache, cu_new, base_len, q, out)


def paged_attn_workspace(d: L.PagedAttnDesc) -> Optional[torch.Tensor]:
    n = L.load().fblt_paged_attn_workspace(C.byref(d))
    return torch.empty(n, dtype=torch.uint8, device=d.keep[0].k_codes.device) if n else None


def paged_attn(d: L.PagedAttnDesc, workspace: Optional[torch.Tensor] = None, stream=None) -> None:
    if workspace is not None and not (workspace.is_cuda and workspace.device.index == d.device and workspace.is_contiguous()):
        raise ValueError(f"workspace: a contiguous tensor on device {d.device} is needed")
    wp = workspace.data_ptr() if workspace is not None else None
    wn = workspace.numel() * workspace.element_size() if workspace is not None else 0
    L.check(L.load().fblt_paged_attn(C.byref(d), wp, wn, _stream_on(d, stream)))


class PagedStepPlan:
    """The self-attention block of a step over the paged cache with every buffer allocated up front (KvStepPlan's
    counterpart): run() only enqueues launches, so steps can be captured in a CUDA graph and replayed while the caches
    grow. x is the static input [total_rows, E], out the static output; rows are packed by cu_new (device), whose last
    entry is total_rows; max_new / max_len bound the new rows and base_len + new rows over every replay.
    w_qkv packs [E, (num_heads + 2 kv_heads) * head_dim] (q | k | v columns), w_proj [E, E]."""

    def __init__(self, w_qkv: PackedWeights, w_proj: PackedWeights, cache: PagedKvCache, cu_new: torch.Tensor,
                 base_len: torch.Tensor, num_heads: int, total_rows: int, max_new: int, max_len: int, *,
                 q_gain: Optional[torch.Tensor] = None, k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                 block_mode: bool = False, window: int = 0, precision: int = L.PREC_FP32):
        hd, dev = cache.head_dim, cache.k_codes.device
        E, W = num_heads * hd, (num_heads + 2 * cache.num_kv_heads) * hd
        if (w_qkv.K, w_qkv.N) != (E, W) or (w_proj.K, w_proj.N) != (E, E):
            raise ValueError(f"weights must be [{E}, {W}] and [{E}, {E}]")
        new = lambda cols: torch.empty(total_rows, cols, dtype=torch.float32, device=dev)  # noqa: E731
        self.x, self.out, self._qkv, self._comb = torch.zeros(total_rows, E, dtype=torch.float32, device=dev), new(E), new(W), new(E)
        a = make_paged_attn(cache, cu_new, base_len, self._comb, self.out, num_heads, max_new, max_len, 1.0,
                            block_mode=block_mode, window=window)
        self._ws = paged_attn_workspace(a)
        d = self.desc = L.PagedStepDesc()
        _keep(d, cache, cu_new, base_len, q_gain, k_gain, rope_cos, rope_sin, w_qkv.buf, w_proj.buf)
        d.cache, d.batch, d.num_heads, d.total_rows, d.max_new = cache.desc, cache.batch, num_heads, total_rows, max_new
        d.max_len, d.block_mode, d.window, d.precision = max_len, int(block_mode), window, precision
        d.cu_new, d.base_len = cu_new.data_ptr(), base_len.data_ptr()
        d.input, d.input_stride = self.x.data_ptr(), self.x.stride(0)
        d.packed_qkv, d.packed_proj = w_qkv.buf.data_ptr(), w_proj.buf.data_ptr()
        d.output, d.output_stride = self.out.data_ptr(), self.out.stride(0)
        d.qkv_work, d.combined_work = self._qkv.data_ptr(), self._comb.data_ptr()
        if self._ws is not None:
            d.workspace, d.workspace_bytes = self._ws.data_ptr(), self._ws.numel()
        d.q_gain, d.k_gain, d.eps = _vector(q_gain, hd, "q_gain"), _vector(k_gain, hd, "k_gain"), float(eps)
        _rope(d, rope_cos, rope_sin, hd)

    def run(self, stream=None) -> None:
        L.check(L.load().fblt_paged_self_attention_step(C.byref(self.desc), _stream_on(self.desc, stream)))


# --------------------------------------------------------------------------- host-buffer sessions

class Session:
    """Host-buffer path: inputs and outputs are host arrays (numpy, or pinned torch CPU
    tensors); every call copies host->device, computes, copies back and returns idle."""

    def __init__(self, max_batch: int, num_heads: int, head_dim: int, max_q_rows: int = 0, max_k_rows: int = 0,
                 cache_rows: int = 0, max_new: int = 0):
        self._lib = L.load()
        self._h = C.c_void_p()
        L.check(self._lib.fblt_session_create(C.byref(self._h), max_batch, num_heads, head_dim, max_q_rows,
                                              max_k_rows, cache_rows, max_new))
        self.num_heads, self.head_dim = num_heads, head_dim

    def close(self) -> None:
        if self._h:
            self._lib.fblt_session_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, q, k, v, out, cu_q, cu_k, scale: float, mask: Optional[MaskConfig] = None, *,
                q_stride=None, k_stride=None, v_stride=None, out_stride=None, impl: int = L.IMPL_AUTO,
                precision: int = L.PREC_FP32, wait: bool = True) -> None:
        """q/k/v/out: host arrays; strides in elements (default: the arrays' own row stride).
        wait=False returns once the work is enqueued (the rows come home beside whatever is called
        next on the session); `out` may be read after wait()."""
        def rs(a, s):
            if s is not None:
                return s
            return a.stride(0) if isinstance(a, torch.Tensor) else a.strides[0] // a.itemsize
        cu_q_h = np.ascontiguousarray(np.asarray(cu_q, dtype=np.int32))
        cu_k_h = np.ascontiguousarray(np.asarray(cu_k, dtype=np.int32))
        batch = len(cu_q_h) - 1
        mask = mask or MaskConfig()
        d = L.AttnDesc()
        d.batch, d.num_heads, d.head_dim = batch, self.num_heads, self.head_dim
        d.max_q = int(np.max(np.diff(cu_q_h))) if batch else 0
        d.max_k = int(np.max(np.diff(cu_k_h))) if batch else 0
        d.impl, d.precision = impl, precision
        d.cu_q, d.cu_k = cu_q_h.ctypes.data, cu_k_h.ctypes.data
        d.q, d.q_stride = _ptr(q), rs(q, q_stride)
        d.k, d.k_stride = _ptr(k), rs(k, k_stride)
        d.v, d.v_stride = _ptr(v), rs(v, v_stride)
        d.out, d.out_stride = _ptr(out), rs(out, out_stride)
        d.scale = float(scale)
        tables = mask.host_tables(batch)
        mask.fill(d.mask, tables)
        fn = self._lib.fblt_session_forward if wait else self._lib.fblt_session_forward_async
        L.check(fn(self._h, C.byref(d)))

    def wait(self) -> None:
        L.check(self._lib.fblt_session_wait(self._h))

    def cache_load(self, lens, k_host, v_host, host_seq_stride_rows: int) -> None:
        lens_h = np.ascontiguousarray(np.asarray(lens, dtype=np.int32))
        L.check(self._lib.fblt_session_cache_load(self._h, len(lens_h), lens_h.ctypes.data_as(L.c_i32_p),
                                                  _ptr(k_host), _ptr(v_host), host_seq_stride_rows))

    def decode(self, batch: int, n_new: int, q_new, k_new, v_new, out, scale: float, *, block_mode: bool = False,
               window: int = 0, advance: Optional[int] = None) -> None:
        L.check(self._lib.fblt_session_decode(self._h, batch, n_new, int(block_mode), window, float(scale),
                                              _ptr(q_new), _ptr(k_new), _ptr(v_new), _ptr(out),
                                              n_new if advance is None else advance))

    def decode_steps(self, batch: int, n_new: int, steps: int, q_new, k_new, v_new, out, scale: float, *,
                     in_step_stride: int = 0, out_step_stride: int = 0, block_mode: bool = False, window: int = 0,
                     advance: Optional[int] = None) -> None:
        """`steps` decode steps with known inputs, copies and kernels overlapped (strides in elements)."""
        L.check(self._lib.fblt_session_decode_steps(self._h, batch, n_new, steps, int(block_mode), window, float(scale),
                                                    _ptr(q_new), _ptr(k_new), _ptr(v_new), in_step_stride, _ptr(out),
                                                    out_step_stride, n_new if advance is None else advance))

    def cache_truncate(self, lens) -> None:
        lens_h = np.ascontiguousarray(np.asarray(lens, dtype=np.int32))
        L.check(self._lib.fblt_session_cache_truncate(self._h, len(lens_h), lens_h.ctypes.data_as(L.c_i32_p)))

    def cache_reset(self) -> None:
        L.check(self._lib.fblt_session_cache_reset(self._h))

    def cache_lens(self, batch: int) -> np.ndarray:
        out = np.zeros(batch, dtype=np.int32)
        L.check(self._lib.fblt_session_cache_lens(self._h, out.ctypes.data_as(L.c_i32_p), batch))
        return out
