"""The average bounds of paged_precision tell the arithmetic of the kernels from what it must not lose (planted here, on the
CPU, in a model of it)."""
import math

import pytest
import torch

import paged_precision as A


def cut(x: torch.Tensor) -> torch.Tensor:
    """float64 -> 24 significant bits, towards zero: what the tensor cores keep of a sum."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.trunc(m * 2.0 ** 24), e - 24)


def halves(x: torch.Tensor, planes: int) -> torch.Tensor:
    """x in units of its row's largest value's power of two, below 2^14, in one or two planes of halves."""
    unit = torch.exp2(torch.frexp(x.abs().amax(-1, keepdim=True))[1].double() - 14)
    y = x / unit
    hi = y.half().double()
    return (hi + ((y - hi).half().double() if planes == 2 else 0)) * unit


def model(q, k, v, scale, q_planes=2, p_planes=2, fold=512):
    """One row per head [H, hd] over k / v [L, hd]: cut sums of 16 products, two planes, folded every `fold` keys."""
    H, hd = q.shape
    qq = halves(q, q_planes)
    s = torch.zeros(H, k.shape[0], dtype=torch.float64)
    for d in range(0, hd, 16):
        s = cut(s + qq[:, d:d + 16] @ k[:, d:d + 16].T)
    x = (s * (scale * math.log2(math.e))).float()
    p = torch.exp2(x - x.amax(-1, keepdim=True)).double()
    pp = halves(p, p_planes)
    out, o = torch.zeros(H, hd, dtype=torch.float32), torch.zeros(H, hd, dtype=torch.float64)
    for i, j in enumerate(range(0, k.shape[0], 16)):
        o = cut(o + pp[:, j:j + 16] @ v[j:j + 16])
        if (i + 1) % (fold // 16) == 0:
            out, o = out + o.float(), torch.zeros_like(o)
    return (out + o.float()) / p.float().sum(-1, keepdim=True)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("chunk", [False, True])
def test_bounds_see_a_lost_plane_and_sums_that_are_not_folded(hd, chunk):
    g = torch.Generator().manual_seed(hd)
    L, H, fold = 8192, 8, 512 if chunk else 256
    q, k, v = (torch.randn(n, hd, generator=g) for n in (H, L, L))
    k, v = (x.mul(32).round().clamp(-127, 127).div(32).double() for x in (k, v))
    scale = 1 / math.sqrt(hd)
    want, s = A.exact(q[None], k[:, None], v[:, None], L, scale)
    rms, mean = A.rms_bound(chunk, hd, L, s), A.pull_bound(chunk, hd, L)
    run = lambda vv=v, **kw: model(q.double(), k, vv, scale, **{"fold": fold, **kw})[None]  # noqa: E731
    assert A.ratio(run(), want) < rms
    assert A.ratio(run(q_planes=1), want) > 4 * rms and A.ratio(run(p_planes=1), want) > 4 * rms
    one, _ = A.exact(q[None], k[:, None], v.abs()[:, None], L, scale)
    assert abs(A.pull(run(v.abs()), one)) < mean
    assert -A.pull(run(v.abs(), fold=1 << 20), one) > 1.5 * mean
