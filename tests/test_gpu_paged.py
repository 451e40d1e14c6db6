"""The 8-bit paged KV cache on the GPU: norm + rotation, append, read back, attention of new rows, and the whole step,
against the definitions in 64 bits (tests/paged_ref.py)."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R
from fblt_b200 import lib as L
from fblt_b200 import ops
from gpu_utils import check_guards, guarded_rows

pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "int8"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def tables(n, hd):
    f = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f[None, :]
    return a.cos().float().cuda(), a.sin().float().cuda()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu(lens):
    return i32(np.concatenate([[0], np.cumsum(lens)]).tolist())


def make_cache(seed, fmt, lens, kv, hd, page, *, spare=2, garbage=True, extra_cols=1):
    """A cache whose pages lie in no order; unused pages, slots and exponents hold garbage bytes."""
    g = gen(seed)
    need = [-(-n // page) for n in lens]
    total, cols = sum(need) + spare, max(max(need), 1) + extra_cols
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((len(lens), cols), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    c = ops.PagedKvCache.empty(total, kv, page, hd, table.cuda(), fmt)
    if garbage:
        for t in (c.k_codes, c.v_codes):
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
        for t in (c.k_exp, c.v_exp):
            t.copy_(torch.randint(-128, 128, t.shape, generator=g, device="cuda").to(torch.int8))
    return c


def stored(c, b, n, which):
    """float64 [n, kv, hd] of positions 0 .. n of sequence b (CPU)."""
    codes, exp = (c.k_codes, c.k_exp) if which == "k" else (c.v_codes, c.v_exp)
    t = c.page_table[b, :-(-n // c.page_size)].long()
    x = R.values(codes[t], exp[t], c.fmt)
    return x.permute(0, 2, 1, 3).reshape(-1, c.num_kv_heads, c.head_dim)[:n]


def fill_cache(c, seed, lens, scale=1.0):
    """Puts quantised normal rows at every position of every sequence through fblt_paged_append."""
    g, cols = gen(seed), c.num_kv_heads * c.head_dim
    rows = sum(lens)
    k, v = randn(g, rows, cols) * scale, randn(g, rows, cols)
    ops.paged_append(ops.make_paged_append(c, cu(lens), i32([0] * len(lens)), k, v))
    torch.cuda.synchronize()
    return k, v


def attend(c, new, base, heads, seed, *, block=False, window=0, splits=0, q=None, scale=None, max_new=None, max_len=None, stream=None):
    hd = c.head_dim
    q = randn(gen(seed), sum(new), heads * hd) if q is None else q
    guard, out = guarded_rows(sum(new), heads * hd, float("nan"))
    d = ops.make_paged_attn(c, cu(new), i32(base), q, out, heads, max(new) if max_new is None else max_new,
                            max(b + n for b, n in zip(base, new)) if max_len is None else max_len,
                            1 / math.sqrt(hd) if scale is None else scale, block_mode=block, window=window, splits=splits)
    ws = ops.paged_attn_workspace(d)
    if ws is not None:
        ws.fill_(0xff)  # NaN in every float: what a call reads it must have written
    ops.paged_attn(d, ws, stream)
    torch.cuda.synchronize()
    check_guards(guard, "paged_attn")
    assert L.load().fblt_tcgen05_error() == 0
    return q, out


def check_attention(c, q, out, new, base, heads, *, block=False, window=0, scale=None, missing=()):
    hd, at = c.head_dim, 0
    scale = 1 / math.sqrt(hd) if scale is None else scale
    for b, (n, p) in enumerate(zip(new, base)):
        if n:
            k, v = stored(c, b, p + n, "k"), stored(c, b, p + n, "v")
            for (mb, lo, hi) in missing:
                if mb == b:
                    k[lo:hi] = math.nan
            want, tol = R.attention(q[at:at + n].view(n, heads, hd), k, v, p, np.float32(scale).item(), block, window)
            got = out[at:at + n].view(n, heads, hd).double().cpu()
            bad = ~((got - want).abs() <= tol)
            assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {bad.numel()} outside the bound, worst "
                                   f"{float(((got - want).abs() / tol)[bad].max()):.3g} times it, at {bad.nonzero()[0].tolist()}")
        at += n


# ------------------------------------------------------------------------------------------------ norm + rotation

@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows,heads,kv", [(1, 1, 1), (3, 5, 2), (37, 8, 8), (2500, 2, 1)])
def test_norm_rope(cuda_lib, hd, rows, heads, kv):
    g = gen(rows * hd)
    pad = 4
    buf = randn(g, rows, (heads + kv) * hd + pad) * 3
    q, k = buf[:, :heads * hd], buf[:, heads * hd:(heads + kv) * hd]
    cos, sin = tables(300, hd)
    pos = torch.randint(0, 300, (rows,), generator=g, device="cuda", dtype=torch.int32)
    qg, kg = randn(g, hd), randn(g, hd)
    gq, qo = guarded_rows(rows, heads * hd, float("nan"))
    gk, ko = guarded_rows(rows, kv * hd, float("nan"))
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, k, pos, heads, kv, hd, q_out=qo, k_out=ko, q_gain=qg, k_gain=kg, eps=1e-5,
                                           rope_cos=cos, rope_sin=sin))
    torch.cuda.synchronize()
    check_guards(gq, "q_out")
    check_guards(gk, "k_out")
    eps = np.float32(1e-5).item()
    for x, o, gain, h in ((q, qo, qg, heads), (k, ko, kg, kv)):
        want = R.norm_rope(x.reshape(rows, h, hd), gain, eps, cos, sin, pos.cpu())
        assert ((o.view(rows, h, hd).double().cpu() - want).abs() <= R.norm_rope_tol(want)).all()
    before = buf.clone()  # in place, and the columns beside are left alone
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, k, pos, heads, kv, hd, q_gain=qg, k_gain=kg, eps=1e-5, rope_cos=cos, rope_sin=sin))
    torch.cuda.synchronize()
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(buf[:, -pad:], before[:, -pad:])


def test_norm_rope_parts(cuda_lib):
    """q alone, k alone, norm without rotation, rotation without norm, positions outside the tables, zero rows."""
    g, hd, rows = gen(3), 64, 9
    q, k = randn(g, rows, 3 * hd), randn(g, rows, 2 * hd)
    q[4] = 0
    cos, sin = tables(10, hd)
    pos, status = i32([0, 9, 10, -1, 3, 2**31 - 1, 5, -2**31, 1]), i32([0])
    gain = randn(g, hd)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, None, pos, 3, 0, hd, q_out=qo, rope_cos=cos, rope_sin=sin, status=status))
    ops.qk_norm_rope(ops.make_qk_norm_rope(None, k, None, 0, 2, hd, k_out=ko, k_gain=gain, eps=0.0))
    torch.cuda.synchronize()
    want = R.norm_rope(q.view(rows, 3, hd), None, 0, cos, sin, pos.cpu())
    assert ((qo.view(rows, 3, hd).double().cpu() - want).abs() <= R.norm_rope_tol(want)).all()
    assert torch.equal(qo[[2, 3, 5, 7]], q[[2, 3, 5, 7]]) and int(status) == L.PAGED_BAD_POSITION
    want = R.norm_rope(k.view(rows, 2, hd), gain, 0, None, None, None)
    assert ((ko.view(rows, 2, hd).double().cpu() - want).abs() <= R.norm_rope_tol(want)).all()
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, None, None, 3, 0, hd, q_out=qo, q_gain=gain, eps=1e-6))
    torch.cuda.synchronize()
    assert bool((qo[4] == 0).all())


# ------------------------------------------------------------------------------------------------ append and read back

def rows_with_edges(g, rows, cols, hd):
    """Normal rows of many sizes; zeros, ties, the borders of an exponent, denormals and the largest values among them."""
    x = randn(g, rows, cols) * torch.pow(10.0, torch.randint(-12, 12, (rows, 1), generator=g, device="cuda").float())
    edge = [0.0, -0.0, 127.0, 127.5, 128.0, 448.0, 449.0, 2.0 ** -126, 1e-40, -1e-45, 3.4e38, -3.4e38, 0.5, 1.5, 2.5, -0.5]
    for i, v in enumerate(edge[:rows]):
        x[i, : hd] = 0
        x[i, i % hd] = v
    if rows > 20:
        x[17, :hd] = torch.arange(hd, device="cuda") + 0.5       # int8 ties under 127
        x[17, 0] = 127.0
        x[18, :hd] = (torch.arange(hd, device="cuda") + 16.5) * 2.0 ** -3
        x[18, 0] = 448.0
        x[19, :hd] = (torch.arange(hd, device="cuda") - 7.5) * 2.0 ** -10  # e4m3's subnormal grid and its ties
        x[19, 0] = 300.0
    return x


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,kv,page,new,base", [
    (32, 1, 16, [1], [0]), (64, 3, 16, [21, 0, 1, 17], [0, 5, 15, 16]), (128, 2, 48, [30, 5], [40, 95]), (64, 2, 1024, [25], [1010])])
def test_append_quantises_exactly_and_reads_back(cuda_lib, fmt, hd, kv, page, new, base):
    g = gen(hd + kv)
    lens = [b + n for b, n in zip(base, new)]
    c = make_cache(1, fmt, lens, kv, hd, page)
    before = [t.clone() for t in (c.k_codes, c.v_codes, c.k_exp, c.v_exp)]
    rows = sum(new)
    k, v = rows_with_edges(g, rows, kv * hd, hd), rows_with_edges(g, rows, kv * hd, hd).flip(0).contiguous()
    ops.paged_append(ops.make_paged_append(c, cu(new), i32(base), k, v))
    torch.cuda.synchronize()
    assert c.status_bits() == 0
    touched = torch.zeros(c.num_pages, kv, page, dtype=torch.bool, device="cuda")
    for x, codes, exp in ((k, c.k_codes, c.k_exp), (v, c.v_codes, c.v_exp)):
        wc, we = R.quantise(x.double().cpu().numpy().reshape(-1, hd), fmt)
        wc, we = wc.reshape(rows, kv, hd), we.reshape(rows, kv)
        r = 0
        for b, (n, p) in enumerate(zip(new, base)):
            for i in range(n):
                pg, slot = int(c.page_table[b, (p + i) // page]), (p + i) % page
                touched[pg, :, slot] = True
                assert (exp[pg, :, slot].cpu().numpy() == we[r]).all(), f"row {r}"
                assert (codes[pg, :, slot].cpu().numpy() == wc[r]).all(), f"row {r}"
                r += 1
    for t, was in zip((c.k_codes, c.v_codes, c.k_exp, c.v_exp), before):
        assert torch.equal(t[~touched], was[~touched]), "slots of other positions changed"
    for dtype in (torch.float32, torch.bfloat16):
        ko, vo = (torch.full((rows + 2, kv * hd + 8), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        ops.paged_read(ops.make_paged_read(c, cu(new), ko[1:-1, :kv * hd], vo[1:-1, :kv * hd], start=i32(base)))
        torch.cuda.synchronize()
        r = 1
        for b, (n, p) in enumerate(zip(new, base)):
            for o, w in ((ko, "k"), (vo, "v")):
                want = stored(c, b, p + n, w)[p:].flatten(1)
                assert torch.equal(o[r:r + n, :kv * hd].double().cpu(), want), f"sequence {b} {w} {dtype}"
            r += n
        for o in (ko, vo):
            assert bool((o[0] == 7).all() and (o[-1] == 7).all() and (o[:, kv * hd:] == 7).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv", [(32, 4, 2), (64, 6, 2), (128, 3, 3)])
def test_append_with_norm_and_rotation(cuda_lib, fmt, hd, heads, kv):
    new, base, page = [5, 0, 33, 1], [11, 3, 0, 63], 32
    g, rows = gen(hd), sum(new)
    c = make_cache(2, fmt, [b + n for b, n in zip(base, new)], kv, hd, page)
    qkv = randn(g, rows, (heads + 2 * kv) * hd)
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
    cos, sin = tables(64, hd)
    qg, kg = 1 + 0.3 * randn(g, hd), 1 + 0.3 * randn(g, hd)
    was = qkv.clone()
    ops.paged_append(ops.make_paged_append(c, cu(new), i32(base), k, v, q=q, num_heads=heads, q_gain=qg, k_gain=kg, eps=1e-6,
                                           rope_cos=cos, rope_sin=sin))  # q in place
    torch.cuda.synchronize()
    assert c.status_bits() == 0 and torch.equal(qkv[:, heads * hd:], was[:, heads * hd:])
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(base, new)])
    eps = np.float32(1e-6).item()
    wq = R.norm_rope(was[:, :heads * hd].reshape(rows, heads, hd), qg, eps, cos, sin, pos)
    assert ((q.reshape(rows, heads, hd).double().cpu() - wq).abs() <= R.norm_rope_tol(wq)).all()
    wk = R.norm_rope(was[:, heads * hd:(heads + kv) * hd].reshape(rows, kv, hd), kg, eps, cos, sin, pos)
    wv = was[:, (heads + kv) * hd:].reshape(rows, kv, hd).double().cpu()
    kc, ke = R.quantise(wk.numpy().reshape(-1, hd), fmt)  # the definition's codes: K goes through 64 bits
    kc, ke = kc.reshape(rows, kv, hd), ke.reshape(rows, kv)
    r = 0
    for b, (n, p) in enumerate(zip(new, base)):
        for i in range(n):
            pg, slot = int(c.page_table[b, (p + i) // page]), (p + i) % page
            assert (c.k_codes[pg, :, slot].cpu().numpy() == kc[r + i]).all() and (c.k_exp[pg, :, slot].cpu().numpy() == ke[r + i]).all()
        for want, codes, exp, tol in ((wk, c.k_codes, c.k_exp, R.norm_rope_tol(wk)), (wv, c.v_codes, c.v_exp, torch.zeros_like(wv))):
            for i in range(n):
                pg, slot = int(c.page_table[b, (p + i) // page]), (p + i) % page
                e = exp[pg, :, slot].cpu().double()[:, None]
                got, x, t = R.values(codes[pg, :, slot], exp[pg, :, slot], fmt), want[r + i], tol[r + i]
                amax = x.abs().amax(-1, keepdim=True)
                assert (amax <= R.QMAX[fmt] * 2 ** e * (1 + 2.0 ** -19)).all() and (amax > R.QMAX[fmt] * 2 ** (e - 1) * (1 - 2.0 ** -19)).all()
                half = torch.maximum((x.abs() + t) * 2.0 ** -4, 2 ** (e - 10)) if fmt == "e4m3" else 2 ** (e - 1)
                assert ((got - x).abs() <= half + t).all()
        r += n


@pytest.mark.parametrize("fmt", FMTS)
def test_append_of_values_that_are_not_finite(cuda_lib, fmt):
    c = make_cache(3, fmt, [4], 1, 32, 16, garbage=False)
    k, v = randn(gen(1), 4, 32), randn(gen(2), 4, 32)
    k[1, 3], k[1, 4], k[1, 5], v[2, :] = math.nan, math.inf, -math.inf, math.nan
    ops.paged_append(ops.make_paged_append(c, cu([4]), i32([0]), k, v))
    torch.cuda.synchronize()
    assert c.status_bits() == L.PAGED_NONFINITE and c.status_bits() == 0
    for x, codes, exp in ((k, c.k_codes, c.k_exp), (v, c.v_codes, c.v_exp)):
        wc, we = R.quantise(x.double().cpu().numpy(), fmt)
        pg = int(c.page_table[0, 0])
        assert (codes[pg, 0, :4].cpu().numpy() == wc).all() and (exp[pg, 0, :4].cpu().numpy() == we).all()


def test_read_of_every_byte(cuda_lib):
    """All 256 codes under the smallest and largest exponents; a range that starts inside a page; K or V alone."""
    for fmt in FMTS:
        lo, hi = R.ELIM[fmt]
        c = make_cache(4, fmt, [32], 2, 64, 16)
        c.k_codes.copy_(torch.arange(256, device="cuda", dtype=torch.uint8).repeat(c.k_codes.numel() // 256).view_as(c.k_codes))
        c.k_exp.copy_(torch.tensor([lo, hi, 0, -8], dtype=torch.int8, device="cuda").repeat(c.k_exp.numel() // 4).view_as(c.k_exp))
        o = torch.full((21, 128), math.nan, device="cuda")
        ops.paged_read(ops.make_paged_read(c, cu([21]), o, None, start=i32([11])))
        torch.cuda.synchronize()
        want = stored(c, 0, 32, "k")[11:].flatten(1)
        # -128 * 2^121 passes fp32's range and the e4m3 codes 0x7f / 0xff are NaN; the library writes none of them
        big = (want.abs() > 3.3e38) | ((want.abs() == 480 * 2.0 ** torch.floor(torch.log2(want.abs() / 256))) & (fmt == "e4m3"))
        assert torch.equal(torch.where(big, 0.0, o.double().cpu()), torch.where(big, 0.0, want))


def test_bad_pages_and_lengths_are_reported(cuda_lib):
    """Page ids outside the pool, positions beyond the table, lengths that describe nothing: no access, a status bit."""
    for fmt in FMTS:
        c = make_cache(5, fmt, [64, 64, 64], 2, 64, 16, extra_cols=0)
        fill_cache(c, 6, [64, 64, 64])
        c.page_table[0, 1], c.page_table[1, 3] = c.num_pages, -1
        codes = c.k_codes.clone()
        k, v = randn(gen(7), 9, 128), randn(gen(8), 9, 128)
        # rows of sequence 0 on its bad page, of sequence 1 across its good / bad border, of sequence 2 past the table
        ops.paged_append(ops.make_paged_append(c, cu([3, 4, 2]), i32([20, 46, 63]), k, v))
        torch.cuda.synchronize()
        assert c.status_bits() == L.PAGED_BAD_PAGE
        wrote = (codes != c.k_codes).flatten(1).any(1)
        wrote = set(wrote.nonzero().flatten().tolist())
        assert wrote == {int(c.page_table[1, 2]), int(c.page_table[2, 3])}
        o = torch.full((40, 128), math.nan, device="cuda")
        ops.paged_read(ops.make_paged_read(c, cu([40, 0, 0]), o, None))
        torch.cuda.synchronize()
        assert c.status_bits() == L.PAGED_BAD_PAGE and bool((o[16:32] == 0).all())
        assert torch.equal(o[:16].double().cpu(), stored(c, 0, 16, "k").reshape(16, -1))
        # attention does not see the keys of such pages
        new, base = [2, 1, 3], [50, 62, 61]
        q, out = attend(c, new, base, 4, 9)
        assert c.status_bits() == L.PAGED_BAD_PAGE
        c.page_table[0, 1] = c.page_table[1, 3] = 0  # any page, for the reference's look-up; its keys are marked missing
        check_attention(c, q, out, new, base, 4, missing=[(0, 16, 32), (1, 48, 64)])
        for tables_ in ((cu([2, 1, 3]), i32([-1, 62, 61])), (i32([0, 2, 1, 3]), i32([50, 62, 61])), (i32([0, 2, 3, 99]), i32([50, 62, 61])),
                        (cu([2, 1, 3]), i32([2**31 - 2, 62, 61]))):
            guard, out = guarded_rows(6, 256, 5.0)
            d = ops.make_paged_attn(c, tables_[0], tables_[1], randn(gen(1), 6, 256), out, 4, 3, 64, 0.125)
            ops.paged_attn(d, ops.paged_attn_workspace(d))
            kk = randn(gen(2), 6, 128)
            ops.paged_append(ops.make_paged_append(c, tables_[0], tables_[1], kk, kk))
            torch.cuda.synchronize()
            check_guards(guard, "bad lengths")
            assert c.status_bits() & L.PAGED_BAD_LENGTH


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (8, 1)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_attention_of_one_token(cuda_lib, fmt, hd, heads, kv, splits):
    base = [0, 1, 15, 16, 127, 128, 300, 1000]
    new = [1] * len(base)
    c = make_cache(10, fmt, [b + 1 for b in base], kv, hd, 16)
    fill_cache(c, 11, [b + 1 for b in base])
    q, out = attend(c, new, base, heads, 12, splits=splits)
    assert c.status_bits() == 0
    check_attention(c, q, out, new, base, heads)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv,page", [(64, 4, 4, 16), (64, 8, 2, 48), (128, 4, 1, 32), (32, 2, 2, 16)])
@pytest.mark.parametrize("new,base", [([2, 3, 0, 8], [0, 30, 5, 200]), ([5, 17, 32], [511, 1, 64]), ([33, 64, 1], [0, 129, 700])])
@pytest.mark.parametrize("block,window", [(False, 0), (True, 0), (False, 1), (False, 40)])
def test_attention_of_a_few_rows(cuda_lib, fmt, hd, heads, kv, page, new, base, block, window):
    lens = [b + n for b, n in zip(base, new)]
    c = make_cache(20, fmt, lens, kv, hd, page)
    fill_cache(c, 21, lens)
    q, out = attend(c, new, base, heads, 22, block=block, window=window)
    check_attention(c, q, out, new, base, heads, block=block, window=window)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("heads,kv,new,base,window,splits", [
    (2, 2, [128], [0], 0, 0), (2, 1, [129, 0, 255], [1, 9, 640], 0, 0), (4, 4, [300, 70], [77, 1000], 0, 2),
    (3, 1, [200, 513], [50, 0], 130, 0), (8, 2, [260], [1500], 0, 0), (5, 1, [97, 150], [33, 260], 97, 3)])
def test_attention_of_a_chunk(cuda_lib, fmt, hd, heads, kv, new, base, window, splits):
    lens = [b + n for b, n in zip(base, new)]
    c = make_cache(30, fmt, lens, kv, hd, 48)
    fill_cache(c, 31, lens)
    q, out = attend(c, new, base, heads, 32, window=window, splits=splits)
    check_attention(c, q, out, new, base, heads, window=window)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [1, 7, 260])
def test_attention_with_keys_and_values_of_very_unequal_size(cuda_lib, fmt, n):
    """Rows whose exponents differ by up to 2^40 beside each other, and scores up to hundreds."""
    hd, heads, kv, base = 64, 4, 2, 300
    c = make_cache(40, fmt, [base + n], kv, hd, 16)
    g = gen(41)
    k, v = randn(g, base + n, kv * hd), randn(g, base + n, kv * hd)
    k *= torch.pow(2.0, torch.randint(-20, 3, (base + n, 1), generator=g, device="cuda").float())
    v *= torch.pow(2.0, torch.randint(-20, 20, (base + n, 1), generator=g, device="cuda").float())
    ops.paged_append(ops.make_paged_append(c, cu([base + n]), i32([0]), k, v))
    q = randn(g, n, heads * hd) * 8
    q, out = attend(c, [n], [base], heads, 0, q=q)
    check_attention(c, q, out, [n], [base], heads)


@pytest.mark.parametrize("n", [1, 5, 200])
def test_queries_that_are_not_finite_or_extreme(cuda_lib, n):
    """Scores that are not finite weigh 0: such a row gives zeros and no other row changes. Very small and very large
    queries are ordinary ones."""
    hd, base = 64, 150
    c = make_cache(50, "e4m3", [base + n], 1, hd, 16)
    fill_cache(c, 51, [base + n])
    q = randn(gen(52), n, 2 * hd)
    clean, was = attend(c, [n], [base], 2, 0, q=q.clone())
    q[0, 3], q[n // 2, hd + 9] = math.inf, math.nan
    _, out = attend(c, [n], [base], 2, 0, q=q)
    assert bool((out[0, :hd] == 0).all()) and bool((out[n // 2, hd:] == 0).all())
    was[0, :hd], was[n // 2, hd:] = 0, 0
    assert torch.equal(out, was)
    for size in (1e-30, 1e-42, 1e30):
        q2, out2 = attend(c, [n], [base], 2, 0, q=clean * size, scale=1e-30 if size > 1 else 0.125)
        check_attention(c, q2, out2, [n], [base], 2, scale=1e-30 if size > 1 else 0.125)


@pytest.mark.parametrize("fmt", FMTS)
def test_result_does_not_depend_on_the_cut_into_chunks(cuda_lib, fmt):
    """A prompt taken at once, in chunks and token by token: the same rows within the bound, the same cache bit for bit."""
    hd, heads, kv, T = 64, 4, 2, 311
    g = gen(60)
    q, k, v = randn(g, T, heads * hd), randn(g, T, kv * hd), randn(g, T, kv * hd)
    outs, caches = [], []
    for cuts in ([T], [100, 1, 77, 133], [1] * 20 + [291]):
        c = make_cache(61, fmt, [T], kv, hd, 16)
        at, out = 0, torch.empty(T, heads * hd, device="cuda")
        for n in cuts:
            ops.paged_append(ops.make_paged_append(c, cu([n]), i32([at]), k[at:at + n], v[at:at + n]))
            _, o = attend(c, [n], [at], heads, 0, q=q[at:at + n])
            out[at:at + n] = o
            at += n
        check_attention(c, q, out, [T], [0], heads)
        outs.append(out)
        caches.append([stored(c, 0, T, w) for w in "kv"])
    for x in caches[1:]:
        assert torch.equal(x[0], caches[0][0]) and torch.equal(x[1], caches[0][1])


def test_shared_pages_and_a_batch_of_copies(cuda_lib):
    """Two sequences whose tables share the pages of a prefix get what copies of them get; the same call twice gives
    the same bits."""
    hd, heads, kv, n = 128, 4, 2, 3
    c = make_cache(70, "int8", [96 + n, 96 + n], kv, hd, 32)
    fill_cache(c, 71, [96 + n, 96 + n])
    c.page_table[1, :3] = c.page_table[0, :3]
    q, out = attend(c, [n, n], [96, 96], heads, 72)
    check_attention(c, q, out, [n, n], [96, 96], heads)
    _, again = attend(c, [n, n], [96, 96], heads, 72)
    assert torch.equal(out, again)


def test_offsets_beyond_32_bits(cuda_lib):
    """Pages whose codes lie past 4 GiB of the pool."""
    hd, kv, page, heads, n = 128, 8, 256, 8, 200
    pages = (1 << 32) // (kv * page * hd) + 8
    for last in (False, True):
        table = i32([[pages - 1, pages - 2, 3, pages - 3] if last else [2, 1, 0, 3]])
        c = ops.PagedKvCache.empty(pages, kv, page, hd, table, "e4m3")
        fill_cache(c, 80, [900])
        for new, base in (([1], [899]), ([n], [700])):
            q, out = attend(c, new, base, heads, 81)
            check_attention(c, q, out, new, base, heads)
        o = torch.empty(900, kv * hd, device="cuda")
        ops.paged_read(ops.make_paged_read(c, cu([900]), None, o))
        torch.cuda.synchronize()
        assert torch.equal(o.double().cpu(), stored(c, 0, 900, "v").reshape(900, -1))
        del c


def test_workspace_is_checked(cuda_lib):
    c = make_cache(90, "e4m3", [4000], 1, 64, 16)
    fill_cache(c, 91, [4000])
    q, out = randn(gen(1), 1, 64), torch.empty(1, 64, device="cuda")
    d = ops.make_paged_attn(c, cu([1]), i32([3999]), q, out, 1, 1, 4000, 0.125, splits=4)
    ws = ops.paged_attn_workspace(d)
    assert ws is not None
    for w in (None, ws[:-16], torch.empty(ws.numel() + 16, dtype=torch.uint8, device="cuda")[8:]):
        with pytest.raises(L.FbltError):
            ops.paged_attn(d, w)
    ops.paged_attn(d, ws)
    torch.cuda.synchronize()
    check_attention(c, q, out, [1], [3999], 1)


def test_more_new_rows_than_announced(cuda_lib):
    """Rows past max_new are left out and reported; the others are right."""
    c = make_cache(92, "int8", [40, 300], 2, 64, 16)
    fill_cache(c, 93, [40, 300])
    for max_new in (2, 130):
        new, base = [2, max_new + 70], [38, 300 - max_new - 70]
        q, out = attend(c, new, base, 2, 94, max_new=max_new)
        assert c.status_bits() == L.PAGED_BAD_LENGTH
        assert bool(torch.isnan(out[2 + max_new:]).all())
        _, whole = attend(c, new, base, 2, 94)
        check_attention(c, q, torch.cat([out[:2 + max_new], whole[2 + max_new:]]), new, base, 2)
        assert c.status_bits() == 0


# ------------------------------------------------------------------------------------------------ together

def make_step(seed, fmt, new, base, heads, kv, hd, page, steps=1, **kw):
    g, E = gen(seed), heads * hd
    W = (heads + 2 * kv) * hd
    total = [b + n * steps for b, n in zip(base, new)]
    c = make_cache(seed, fmt, total, kv, hd, page)
    if sum(base):
        fill_cache(c, seed + 1, base)
    wq, wp = ops.PackedWeights(randn(g, E, W) / math.sqrt(E)), ops.PackedWeights(randn(g, E, E) / math.sqrt(E))
    cos, sin = tables(max(total) + 1, hd)
    gains = dict(q_gain=1 + 0.1 * randn(g, hd), k_gain=1 + 0.1 * randn(g, hd), eps=1e-6, rope_cos=cos, rope_sin=sin)
    bl = i32(base)
    plan = ops.PagedStepPlan(wq, wp, c, cu(new), bl, heads, sum(new), max(new), max(total), **gains, **kw)
    return c, plan, wq, wp, gains, bl


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new,base", [([1, 1, 1], [0, 40, 700]), ([150, 3, 0, 90], [10, 0, 5, 300])])
def test_step_is_its_parts(cuda_lib, fmt, new, base):
    """The block against its parts run one by one: the same bits in the cache and in the output."""
    heads, kv, hd = 4, 2, 64
    c, plan, wq, wp, gains, bl = make_step(100, fmt, new, base, heads, kv, hd, 16)
    c2 = ops.PagedKvCache(c.k_codes.clone(), c.v_codes.clone(), c.k_exp.clone(), c.v_exp.clone(), c.page_table, fmt)
    plan.x.copy_(randn(gen(5), *plan.x.shape))
    plan.run()
    torch.cuda.synchronize()
    E = heads * hd
    qkv = ops.matmul(plan.x, wq)
    q, k, v = qkv[:, :E], qkv[:, E:E + kv * hd], qkv[:, E + kv * hd:]
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, None, torch.cat([torch.arange(b, b + n, device="cuda", dtype=torch.int32) for b, n in zip(base, new)]),
                                           heads, kv, hd, q_gain=gains["q_gain"], eps=1e-6, rope_cos=gains["rope_cos"], rope_sin=gains["rope_sin"]))
    ops.paged_append(ops.make_paged_append(c2, cu(new), bl, k, v, k_gain=gains["k_gain"], eps=1e-6, rope_cos=gains["rope_cos"],
                                           rope_sin=gains["rope_sin"]))
    for a, b in ((c.k_codes, c2.k_codes), (c.v_codes, c2.v_codes), (c.k_exp, c2.k_exp), (c.v_exp, c2.v_exp)):
        assert torch.equal(a, b)
    _, comb = attend(c2, new, base, heads, 0, q=q, max_len=max(b + n for b, n in zip(base, new)))
    check_attention(c2, q, comb, new, base, heads)
    assert torch.equal(plan.out, ops.matmul(comb, wp))


def test_steps_replayed_from_graphs_on_their_own_streams(cuda_lib):
    """Two plans over two caches, each captured on a stream of its own, replayed at the same time while the lengths grow
    on the device; what a plan launched from the host gives, bit for bit."""
    heads, kv, hd, steps = 4, 2, 64, 6
    runs = []
    for seed, new, base in ((110, [1, 1], [20, 333]), (120, [3, 0, 2], [0, 7, 90])):
        c, plan, wq, wp, gains, bl = make_step(seed, "e4m3", new, base, heads, kv, hd, 16, steps=steps)
        xs = randn(gen(seed + 9), steps, *plan.x.shape)
        saved = [t.clone() for t in (c.k_codes, c.v_codes, c.k_exp, c.v_exp)]
        want = []
        for t in range(steps):
            plan.x.copy_(xs[t])
            plan.run()
            want.append(plan.out.clone())
            bl += i32(new)
        torch.cuda.synchronize()
        for t, s in zip((c.k_codes, c.v_codes, c.k_exp, c.v_exp), saved):
            t.copy_(s)
        bl.copy_(i32(base))
        xin, tin, outs = xs.clone(), torch.zeros(1, dtype=torch.long, device="cuda"), torch.zeros(steps, *plan.out.shape, device="cuda")
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        inc = i32(new)
        with torch.cuda.graph(graph, stream=stream):
            plan.x.copy_(xin.index_select(0, tin)[0])
            plan.run()
            outs.index_copy_(0, tin, plan.out[None])
            bl += inc
            tin += 1
        runs.append((stream, graph, outs, torch.stack(want), (c, plan, wq, wp, gains, bl, xin, tin, inc)))
    torch.cuda.synchronize()
    for _ in range(steps):
        for stream, graph, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, graph, outs, want, _ in runs:
        assert torch.equal(outs, want)
        graph.reset()


def test_on_another_stream(cuda_lib):
    c = make_cache(130, "int8", [500], 2, 64, 16)
    fill_cache(c, 131, [500])
    q, want = attend(c, [200], [300], 4, 132)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    _, got = attend(c, [200], [300], 4, 0, q=q, stream=s)
    assert torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 20, 150])
def test_lengths_far_beyond_the_page_table(cuda_lib, n):
    """A length near 2^31: nothing walks past the table; the keys that exist are attended to and the rest is reported."""
    c = make_cache(150, "int8", [64], 2, 64, 16, extra_cols=0)
    fill_cache(c, 151, [64])
    base = 2**31 - 1 - n - 5000
    q, out = attend(c, [n], [base], 4, 152, max_len=4096)
    assert c.status_bits() == L.PAGED_BAD_PAGE
    k, v = stored(c, 0, 64, "k"), stored(c, 0, 64, "v")
    want, tol = R.attention(q.view(n, 4, 64), k, v, 10**6, 0.125, False, 0)
    assert ((out.view(n, 4, 64).double().cpu() - want).abs() <= tol).all()
    _, out = attend(c, [n], [base], 4, 152, max_len=4096, window=100)  # a window that has left the table
    assert bool((out == 0).all()) and c.status_bits() == L.PAGED_BAD_PAGE


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n", [1, 200])
def test_rows_of_zeros_and_of_the_smallest_values(cuda_lib, fmt, n):
    """Zeros in K and V between ordinary rows, and caches whose every value lies near the smallest exponent."""
    hd, kv, base = 64, 2, 250
    for size in (1.0, 2.0 ** -119, 2.0 ** -90):
        c = make_cache(160, fmt, [base + n], kv, hd, 16)
        g = gen(161)
        k, v = randn(g, base + n, kv * hd) * size, randn(g, base + n, kv * hd) * size
        k[::7], v[::5] = 0, 0
        ops.paged_append(ops.make_paged_append(c, cu([base + n]), i32([0]), k, v))
        q = randn(g, n, 4 * hd) / size
        q, out = attend(c, [n], [base], 4, 0, q=q)
        check_attention(c, q, out, [n], [base], 4)


def test_two_calls_at_once(cuda_lib):
    """The same kernels on two streams at the same time, each with its own workspace and status."""
    jobs = []
    for seed, new, base in ((170, [1, 1], [900, 3000]), (171, [300], [2000])):
        c = make_cache(seed, "e4m3", [b + n for b, n in zip(base, new)], 2, 64, 32)
        fill_cache(c, seed + 5, [b + n for b, n in zip(base, new)])
        q = randn(gen(seed), sum(new), 4 * 64)
        out = torch.empty_like(q)
        d = ops.make_paged_attn(c, cu(new), i32(base), q, out, 4, max(new), 3100, 0.125, splits=3)
        jobs.append((d, ops.paged_attn_workspace(d), torch.cuda.Stream(), c, q, out, new, base))
    torch.cuda.synchronize()
    for _ in range(20):
        for d, ws, s, *_ in jobs:
            ops.paged_attn(d, ws, s)
    torch.cuda.synchronize()
    for d, ws, s, c, q, out, new, base in jobs:
        check_attention(c, q, out, new, base, 4)


def test_bindings_refuse_wrong_tensors(cuda_lib):
    c = make_cache(140, "e4m3", [32], 2, 64, 16)
    k = torch.zeros(4, 128, device="cuda")
    bad = [dict(k=k.double()), dict(k=k[:, :64]), dict(v=k.cpu()), dict(v=k[:2]), dict(q=k, num_heads=4), dict(k_gain=k[0, :32])]
    for b in bad:
        a = dict(k=k, v=k)
        a.update(b)
        with pytest.raises(ValueError):
            ops.make_paged_append(c, cu([4]), i32([0]), a.pop("k"), a.pop("v"), **a)
    with pytest.raises(ValueError):
        ops.make_paged_append(c, cu([4]).long(), i32([0]), k, k)
    with pytest.raises(ValueError):
        ops.make_paged_read(c, cu([4]), k, k.bfloat16())
    with pytest.raises(ValueError):
        ops.PagedKvCache(c.k_codes, c.v_codes, c.k_exp.float(), c.v_exp, c.page_table, "e4m3")
    d = ops.make_paged_append(c, cu([4]), i32([0]), k, k)
    d.device = 1  # as if the tensors were on another device than the current one
    with pytest.raises(ValueError):
        ops.paged_append(d)


# ------------------------------------------------------------------------------------------------ long launches

@pytest.mark.parametrize("hd,heads,kv,rows", [(32, 1, 1, 4001), (64, 16, 4, 7301), (128, 5, 3, 3600), (64, 2, 7, 15000)])
def test_a_long_launch_gives_what_short_ones_give(cuda_lib, hd, heads, kv, rows):
    """CTAs that take several rows and share heads and rows among their threads: the bits of launches of a row a CTA."""
    g = gen(rows)
    cuts = np.unique(np.concatenate([[0, rows], np.random.default_rng(rows).integers(1, rows, 23)]))
    new = np.diff(cuts).tolist()
    base = [7 * b % 50 for b in range(len(new))]
    caches = [make_cache(95, "int8", [b + n for b, n in zip(base, new)], kv, hd, 16) for _ in range(2)]
    qkv = randn(g, rows, (heads + 2 * kv) * hd)
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
    cos, sin = tables(4000, hd)  # some positions lie outside of them
    gain = 1 + 0.3 * randn(g, hd)
    outs = [torch.full((rows + 2, heads * hd), 7.0, device="cuda") for _ in range(2)]

    def append(c, lo, hi, out):  # sequences lo .. hi
        a, b = int(cuts[lo]), int(cuts[hi])
        part = ops.PagedKvCache(c.k_codes, c.v_codes, c.k_exp, c.v_exp, c.page_table[lo:hi], c.fmt)
        ops.paged_append(ops.make_paged_append(part, cu(new[lo:hi]), i32(base[lo:hi]), k[a:b], v[a:b], q=q[a:b], num_heads=heads,
                                               q_out=out[1 + a:1 + b], q_gain=gain, k_gain=gain, eps=1e-6, rope_cos=cos, rope_sin=sin))

    append(caches[0], 0, len(new), outs[0])
    for i in range(len(new)):
        append(caches[1], i, i + 1, outs[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and bool((outs[0][0] == 7).all() and (outs[0][-1] == 7).all())
    for name in ("k_codes", "v_codes", "k_exp", "v_exp"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    c = caches[0]
    ko, vo = (torch.full((rows + 2, kv * hd), 7.0, device="cuda") for _ in range(2))
    ops.paged_read(ops.make_paged_read(c, cu(new), ko[1:-1], vo[1:-1], start=i32(base)))
    only = torch.full((rows + 2, kv * hd), 7.0, device="cuda")
    ops.paged_read(ops.make_paged_read(c, cu(new), None, only[1:-1], start=i32(base)))
    torch.cuda.synchronize()
    assert torch.equal(vo, only)
    for o, w in ((ko, "k"), (vo, "v")):
        want = torch.cat([stored(c, b, p + n, w)[p:].flatten(1) for b, (n, p) in enumerate(zip(new, base))])
        assert torch.equal(o[1:-1].double().cpu(), want) and bool((o[0] == 7).all() and (o[-1] == 7).all())
    pos = torch.randint(-5, 4100, (rows,), generator=g, device="cuda", dtype=torch.int32)
    long, short = torch.empty(rows, heads * hd, device="cuda"), torch.empty(rows, heads * hd, device="cuda")
    ops.qk_norm_rope(ops.make_qk_norm_rope(q, None, pos, heads, 0, hd, q_out=long, q_gain=gain, eps=1e-6, rope_cos=cos, rope_sin=sin))
    for a in range(0, rows, 1000):
        b = min(rows, a + 1000)
        ops.qk_norm_rope(ops.make_qk_norm_rope(q[a:b], None, pos[a:b], heads, 0, hd, q_out=short[a:b], q_gain=gain, eps=1e-6,
                                               rope_cos=cos, rope_sin=sin))
    torch.cuda.synchronize()
    assert torch.equal(long, short)


@pytest.mark.parametrize("hd,n", [(128, 1), (128, 3), (128, 8), (64, 6), (64, 8), (32, 8)])
@pytest.mark.parametrize("step", [0.02, 0.4])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_rise_or_fall_slowly(cuda_lib, hd, n, step, falling):
    """Every key a little above the one before it (a maximum that grows by less than the rescaling waits for), or below."""
    heads, kv, base = 4, 1, 700
    L_ = base + n
    c = make_cache(97, "int8", [L_], kv, hd, 16)
    u = torch.ones(hd, device="cuda")
    ramp = torch.arange(L_, device="cuda").float() * step / hd
    k = (ramp.flip(0) if falling else ramp)[:, None] * u
    v = randn(gen(98), L_, hd)
    ops.paged_append(ops.make_paged_append(c, cu([L_]), i32([0]), k.contiguous(), v))
    q = u.repeat(heads)[None, :] * (1 + 0.1 * torch.arange(n, device="cuda").float()[:, None])
    for splits in (1, 3):
        _, out = attend(c, [n], [base], heads, 0, q=q.contiguous(), scale=1.0, splits=splits)
        check_attention(c, q, out, [n], [base], heads, scale=1.0)


@pytest.mark.parametrize("hd,heads,kv,batch,new,max_len", [
    (128, 32, 8, 75, 8, 8192), (64, 16, 4, 160, 5, 12000), (64, 8, 4, 41, 300, 4096)])
def test_many_short_sequences_in_a_launch_planned_for_long_ones(cuda_lib, hd, heads, kv, batch, new, max_len):
    """Pieces without a key, and tiles that are not split: the plan follows max_len and the batch, not the lengths."""
    base = [(37 * b) % 200 for b in range(batch)]
    news = [new if b % 3 else new // 2 for b in range(batch)]
    lens = [b + n for b, n in zip(base, news)]
    c = make_cache(99, "e4m3", lens, kv, hd, 32)
    fill_cache(c, 100, lens)
    q, out = attend(c, news, base, heads, 101, max_new=new, max_len=max_len)
    assert c.status_bits() == 0
    check_attention(c, q, out, news, base, heads)
