"""The paged cache's operators where they could go wrong between calls of their ordinary tests: pieces and tiles without
keys, stages that are used again, scales at both ends of fp32, limits of a launch, and precision over long ranges."""
import math

import numpy as np
import pytest
import torch

import paged_precision as A
from fblt_b200 import lib as L
from fblt_b200 import ops
from test_gpu_paged import attend, check_attention, cu, fill_cache, gen, i32, make_cache, randn, stored

pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "int8"]


# ------------------------------------------------------------------------------------------------ pieces without keys

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv", [(32, 8, 2), (64, 8, 2), (128, 8, 2), (64, 2, 2)])
@pytest.mark.parametrize("new,base,splits", [([300, 70, 0, 150], [0, 9, 4, 2100], 8), ([129, 257], [0, 3000], 5)])
def test_queries_that_are_not_finite_beside_pieces_without_keys(cuda_lib, fmt, hd, heads, kv, new, base, splits):
    """A prompt's first rows in a launch cut for a long sequence: most pieces have no key. A query row that is not finite
    gives zeros, and every other row the bits that it has without it."""
    lens = [b + n for b, n in zip(base, new)]
    c = make_cache(200, fmt, lens, kv, hd, 48)
    fill_cache(c, 201, lens)
    q = randn(gen(202), sum(new), heads * hd)
    _, want = attend(c, new, base, heads, 0, q=q.clone(), splits=splits)
    bad = q.clone().view(-1, heads, hd)
    where = torch.zeros(sum(new), heads, dtype=torch.bool, device="cuda")
    for r in range(0, sum(new), 3):
        for h in range(heads):
            if (r + h) % 4 == 0:
                bad[r, h, (5 * r + h) % hd] = (math.nan, math.inf, -math.inf)[(r // 3 + h) % 3]
                where[r, h] = True
    for _ in range(5):
        _, got = attend(c, new, base, heads, 0, q=bad.view(-1, heads * hd), splits=splits)
        got = got.view(-1, heads, hd)
        assert bool((got[where] == 0).all())
        assert torch.equal(got[~where], want.view(-1, heads, hd)[~where])
    check_attention(c, q, want, new, base, heads)


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("splits", [1, 4])
def test_a_tile_without_any_key(cuda_lib, hd, splits):
    """Rows whose window has left the page table: zeros, whatever the queries hold."""
    n, heads = 260, 2
    c = make_cache(203, "int8", [64], 2, hd, 16, extra_cols=0)
    fill_cache(c, 204, [64])
    q = randn(gen(205), n, heads * hd)
    q[::5, 3], q[1::7, hd + 1] = math.nan, math.inf
    for _ in range(5):
        _, out = attend(c, [n], [5000], heads, 0, q=q, window=100, splits=splits)
        assert bool((out == 0).all()) and c.status_bits() == L.PAGED_BAD_PAGE


# ------------------------------------------------------------------------------------------------ stages that are used again

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,kv,new", [(32, 4, 1, 5), (64, 4, 1, 6), (64, 8, 2, 8), (128, 4, 2, 6), (128, 4, 1, 4), (128, 4, 1, 8)])
@pytest.mark.parametrize("window", [0, 1003, 2041])
def test_stages_whose_values_were_cleared_are_used_again(cuda_lib, fmt, hd, heads, kv, new, window):
    """Warps that share keys: the first stage of a window and the stages around a missing page hold cleared rows of V, and
    their shared memory takes the keys of later stages, many times over."""
    news, base = [new, new - 1, new], [2500, 2077, 1300]
    lens = [b + n for b, n in zip(base, news)]
    c = make_cache(210, fmt, lens, kv, hd, 16)
    fill_cache(c, 211, lens)
    gone = [(0, 1600, 1616), (0, 1680, 1696), (1, 1200, 1216), (2, 16, 32), (2, 640, 656)]
    keep = c.page_table.clone()
    for b, lo, _ in gone:
        c.page_table[b, lo // 16] = -1
    for _ in range(3):
        q, out = attend(c, news, base, heads, 212, window=window, splits=1)
        assert c.status_bits() == L.PAGED_BAD_PAGE
    c.page_table.copy_(keep)
    check_attention(c, q, out, news, base, heads, window=window, missing=gone)


# ------------------------------------------------------------------------------------------------ large launches

@pytest.mark.parametrize("splits", [0, 2])
def test_single_tokens_of_many_sequences_beside_a_long_chunk(cuda_lib, splits):
    """1100 sequences x 64 tiles of rows, more than a grid's second and third dimension hold."""
    new, heads, kv, hd = [1] * 700 + [2048] + [1] * 399, 8, 1, 32
    base = [(29 * b) % 90 for b in range(len(new))]
    lens = [b + n for b, n in zip(base, new)]
    c = make_cache(220, "int8", lens, kv, hd, 32)
    fill_cache(c, 221, lens)
    q, out = attend(c, new, base, heads, 222, splits=splits)
    assert c.status_bits() == 0
    check_attention(c, q, out, new, base, heads)


# ------------------------------------------------------------------------------------------------ scales at both ends of fp32

def append_all(c, k, v):
    ops.paged_append(ops.make_paged_append(c, cu([k.shape[0]]), i32([0]), k, v))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 5, 20, 150, 300])
@pytest.mark.parametrize("low,high", [(-100, 100), (-107, 120), (-117, 122)])
def test_values_at_both_ends_of_the_range(cuda_lib, fmt, hd, n, low, high):
    """Rows that see only very small values, beside very large ones that the mask or the softmax takes out: first the large
    rows lie behind the small ones (a causal mask), then before them (a window), then among them with weights of 0."""
    if fmt == "e4m3":
        low = max(low, -107)  # 448 * 2^-117 is the largest value of the least exponent
    heads, base = 2, 90
    L_ = base + n
    g = gen(230)
    for where in ("behind", "before", "among"):
        c = make_cache(231, fmt, [L_], 1, hd, 16)
        k, v, q = randn(g, L_, hd), randn(g, L_, hd).clamp(-2, 2), randn(g, n, heads * hd)
        big = torch.zeros(L_, dtype=torch.bool, device="cuda")
        window = 0
        if where == "behind":
            big[base + n // 2 + 1:] = True  # the first half of the new rows sees small values alone
        elif where == "before":
            big[:60], window = True, 31     # (row base sees 60 ..)
        else:
            big[7::16] = True
            u = torch.ones(hd, device="cuda")
            k[big] = -40 * u
            q = (0.9 + 0.2 * torch.rand(q.shape, generator=g, device="cuda"))  # scores of about -40 sqrt(hd): e^-226 or less
        v *= torch.where(big, 2.0 ** high, 2.0 ** low)[:, None]
        append_all(c, k, v)
        for splits in (1, 2):
            q, out = attend(c, [n], [base], heads, 0, q=q, window=window, splits=splits)
            assert c.status_bits() == 0
            check_attention(c, q, out, [n], [base], heads, window=window)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 200])
@pytest.mark.parametrize("every", [16, 128])
def test_small_weights_that_make_up_for_the_size_of_values(cuda_lib, fmt, hd, n, every):
    """Keys of weight 2^-118 or so whose values are 2^120 times the others': both count, whichever tile they lie in."""
    heads, base = 2, 256
    L_ = base + n
    c = make_cache(240, fmt, [L_], 1, hd, 16)
    g = gen(241)
    big = torch.arange(L_, device="cuda") // every % 2 == 1
    k = 0.05 * randn(g, L_, hd)
    k -= torch.where(big, 82.0 / math.sqrt(hd), 0.0)[:, None]
    v = randn(g, L_, hd) * torch.where(big, 2.0 ** 111, 2.0 ** -9)[:, None]
    append_all(c, k, v)
    q = 1 + 0.01 * randn(g, n, heads * hd)
    for splits in (1, 2):
        q, out = attend(c, [n], [base], heads, 0, q=q, splits=splits)
        check_attention(c, q, out, [n], [base], heads)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 6, 15, 150])
def test_keys_at_both_ends_of_the_range(cuda_lib, fmt, hd, n):
    """Scores of ordinary size from very small queries and very large keys, and from very large queries over very small
    keys beside keys whose scores pass fp32 (those weigh 0)."""
    heads, base = 2, 130
    L_ = base + n
    g = gen(250)
    small, large = 2.0 ** -107, 2.0 ** 118
    for keys, queries, over in (("large", 2.0 ** -118, ()), ("small", 2.0 ** 107, ()), ("small", 2.0 ** 107, (3, 16, 17, 60, 128))):
        c = make_cache(251, fmt, [L_], 1, hd, 16)
        k, v, q = randn(g, L_, hd).clamp(-4, 4), randn(g, L_, hd), randn(g, n, heads * hd).clamp(-4, 4)
        k *= large if keys == "large" else small
        for j in over:
            k[j] = k[j] * 2.0 ** 100 * 2.0 ** 100  # (2^200 is no float)
        append_all(c, k, v)
        q *= queries
        for splits in (1, 2):
            q, out = attend(c, [n], [base], heads, 0, q=q, splits=splits)
            assert c.status_bits() == 0
            check_attention(c, q, out, [n], [base], heads, missing=[(0, j, j + 1) for j in over])


@pytest.mark.parametrize("hd", [32, 128])
@pytest.mark.parametrize("n", [1, 6, 15, 150])
def test_scores_that_are_zero_between_scores_that_pass_fp32(cuda_lib, hd, n):
    """One-hot queries and keys of 2^100: a score is 0 or not finite, and the zeros share the weight."""
    heads, base = 2, 100
    L_ = base + n
    c = make_cache(252, "int8", [L_], 1, hd, 16)
    k, q = torch.zeros(L_, hd, device="cuda"), torch.zeros(n, heads * hd, device="cuda")
    hit = torch.arange(L_, device="cuda") % 3 == 1
    k[hit, 2], k[~hit, 5] = 2.0 ** 100, 2.0 ** 100
    q[:, 2::hd] = 2.0 ** 100
    v = randn(gen(253), L_, hd)
    append_all(c, k, v)
    q, out = attend(c, [n], [base], heads, 0, q=q)
    check_attention(c, q, out, [n], [base], heads, missing=[(0, j, j + 1) for j in hit.nonzero().flatten().tolist()])


# ------------------------------------------------------------------------------------------------ precision over long ranges

LONG = [(32, 1, 1), (64, 1, 1), (128, 1, 1), (64, 4, 3), (32, 4, 7), (64, 4, 8), (128, 4, 3), (128, 4, 8), (32, 4, 40), (64, 4, 40), (128, 4, 40)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd,heads,n", LONG)
@pytest.mark.parametrize("sink", [False, True])
def test_average_error_over_long_ranges(cuda_lib, fmt, hd, heads, n, sink):
    """Both planes of Q and P are there, and the sums are folded: averages that a lost one would raise by far
    (test_paged_precision). `sink`: the first keys are small and their values smaller, as a model's first tokens are, so that
    exponents of a tile lie far apart."""
    L_, kv = 8000 + n, 1
    chunk = n * heads // kv > 32
    c = make_cache(260, fmt, [L_], kv, hd, 64)
    g = gen(261)
    k, v, q = randn(g, L_, hd), randn(g, L_, hd), randn(g, n, heads * hd)
    if sink:
        k[:4] *= 2.0 ** -6
        v[:4] *= 2.0 ** -9
    for sign in (False, True):
        append_all(c, k, v.abs() if sign else v)
        _, out = attend(c, [n], [L_ - n], heads, 0, q=q, splits=1)
        kk, vv = stored(c, 0, L_, "k").cuda(), stored(c, 0, L_, "v").cuda()
        want, size = A.exact(q.view(n, heads, hd), kk, vv, L_ - n, np.float32(1 / math.sqrt(hd)).item())
        got = out.view(n, heads, hd)
        if sign:
            pull, bound = A.pull(got, want), A.pull_bound(chunk, hd, L_)
            assert abs(pull) <= bound, f"mean signed error {pull:.3g}, bound {bound:.3g}"
        else:
            r, bound = A.ratio(got, want), A.rms_bound(chunk, hd, L_, size)
            assert r <= bound, f"rms error {r:.3g} of the rms output, bound {bound:.3g}"


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_cuts_into_chunks_agree_on_average(cuda_lib, fmt, hd):
    """A prompt at once, in chunks and token by token: outputs that differ by what their errors allow, no more."""
    heads, kv, T = 4, 2, 311
    g = gen(262)
    q, k, v = randn(g, T, heads * hd), randn(g, T, kv * hd), randn(g, T, kv * hd)
    outs = []
    for cuts in ([T], [100, 1, 77, 133], [1] * 20 + [291], [17] * 18 + [5]):
        c, at, parts = make_cache(263, fmt, [T], kv, hd, 16), 0, []
        for m in cuts:
            ops.paged_append(ops.make_paged_append(c, cu([m]), i32([at]), k[at:at + m], v[at:at + m]))
            parts.append(attend(c, [m], [at], heads, 0, q=q[at:at + m])[1])
            at += m
        outs.append(torch.cat(parts))
    kk, vv = stored(c, 0, T, "k").cuda(), stored(c, 0, T, "v").cuda()
    want, size = A.exact(q.view(T, heads, hd), kk, vv, 0, np.float32(1 / math.sqrt(hd)).item())
    bound = A.rms_bound(True, hd, T, size)
    for o in outs:
        assert A.ratio(o.view(T, heads, hd), want) <= bound
    for o in outs[1:]:
        assert A.ratio(o, outs[0].double()) <= 2 * bound
