"""The paged 8-bit cache operators in 64 bits on the CPU, from their definitions, and the error bounds the tests use."""
from __future__ import annotations

import math

import numpy as np
import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}
ELIM = {"e4m3": (-117, 119), "int8": (-126, 121)}
U24 = 2.0 ** -24


def code_table(fmt: str) -> np.ndarray:
    """The value of every byte."""
    b = np.arange(256)
    if fmt == "int8":
        return np.where(b < 128, b, b - 256).astype(np.float64)
    s, e, m = np.where(b & 128, -1.0, 1.0), (b >> 3) & 15, b & 7
    return s * np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m * 2.0 ** -9)


def values(codes: torch.Tensor, exp: torch.Tensor, fmt: str) -> torch.Tensor:
    """float64 values of codes [..., hd] with exponents [...]."""
    t = torch.from_numpy(code_table(fmt))
    return t[codes.cpu().long()] * torch.pow(torch.tensor(2.0, dtype=torch.float64), exp.cpu().double())[..., None]


def exponent(amax: float, fmt: str) -> int:
    lo, hi = ELIM[fmt]
    e = lo
    while e < hi and amax > QMAX[fmt] * 2.0 ** e:
        e += 1
    return e


def quantise(x: np.ndarray, fmt: str):
    """(codes, exponents) of rows x [n, hd] (float32 values in float64), one row at a time by the definition."""
    table, order = code_table(fmt), None
    ok = np.arange(256) if fmt == "int8" else np.array([b for b in range(256) if b not in (0x7f, 0xff)])
    if fmt == "int8":
        ok = ok[table[ok] >= -127]
    vals = table[ok]
    order = np.argsort(vals, kind="stable")
    vals, ok = vals[order], ok[order]
    codes, exps = np.zeros(x.shape, np.uint8), np.zeros(x.shape[0], np.int8)
    for r, row in enumerate(x):
        fin = np.abs(row[np.isfinite(row)])
        e = exponent(float(fin.max()) if fin.size else 0.0, fmt)
        exps[r] = e
        for i, v in enumerate(row):
            if math.isnan(v):
                continue
            y = min(max(float(v) * 2.0 ** -e, -QMAX[fmt]), QMAX[fmt])
            j = int(np.searchsorted(vals, y))
            cand = [k for k in (j - 1, j, j + 1) if 0 <= k < len(vals)]
            best = min(abs(vals[k] - y) for k in cand)
            near = [k for k in cand if abs(vals[k] - y) == best]
            # a tie goes to the even code; both zeros stand for zero and the sign follows the input
            pick = near[0] if len({vals[k] for k in near}) == 1 else next(k for k in near if (int(ok[k]) & 1) == 0)
            if vals[pick] == 0:
                codes[r, i] = 0x80 if fmt == "e4m3" and math.copysign(1.0, y) < 0 else 0
            else:
                codes[r, i] = ok[pick]
    return codes, exps


def norm_rope(x, gain, eps, cos, sin, pos):
    """x [rows, heads, hd] -> float64; gain, tables may be None. Positions outside the tables leave a row unrotated."""
    x = x.double().cpu()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double().cpu()
    if cos is None:
        return x
    out = x.clone()
    for r in range(x.shape[0]):
        p = int(pos[r])
        if 0 <= p < cos.shape[0]:
            c, s = cos[p].double().cpu(), sin[p].double().cpu()
            out[r, :, 0::2] = x[r, :, 0::2] * c - x[r, :, 1::2] * s
            out[r, :, 1::2] = x[r, :, 1::2] * c + x[r, :, 0::2] * s
    return out


def norm_rope_tol(y: torch.Tensor) -> torch.Tensor:
    """Bound of the fp32 error at y [..., hd] (float64 result). The sum of squares is a tree of at most 9 roundings per
    term, with the mean and eps 11, halved by the root: 5.5 * 2^-24 relative; rsqrt is off by at most 2 units of the last
    place, 4 * 2^-24, and two products round: 11.5 * 2^-24. The rotation adds a product and a sum, 2 * 2^-24 of
    |y0 c| + |y1 s| <= sqrt(2) hypot: 16 * 2^-24 of the pair's length covers both."""
    h = torch.sqrt(y[..., 0::2] ** 2 + y[..., 1::2] ** 2)
    return 16 * U24 * torch.repeat_interleave(h, 2, dim=-1) + 1e-37


def attention(q, k, v, base, scale, block, window):
    """q [n, H, hd], k / v [base + n, KV, hd] (float64; a key that is not there has NaN) -> (out, bound) [n, H, hd].

    The bound, per element, in units of sum_k p_k |v_k|. A weight's relative error is the error of its score: products
    carry 22 bits of q (2^-22 relative), the hd-term sum and its scaling round at most hd + 8 times with at most 2^-23
    each (tensor-core sums truncate), and the largest score is subtracted in the same precision. Numerator and
    denominator carry it both: twice. Weights and values then carry 22 bits, and a sum over L keys is made of at most
    3 L / 8 + 64 additions of 2^-23.

    Weights times V's scales, p 2^e, may be held in halves in units of 2^(R - 10), R at most five above the exponent of
    the row's largest p 2^e (key k*; four for the exponents of a tile that are taken as one, one for rounding a moved
    maximum down): half a step of a half's fixed-point end is 2^-25 of that unit, an error of 2^-30 p* 2^e* in each
    weight and so of 2^-30 p* 2^e* Qmax in its product with a code. The largest |v| of row k* is at least Qmax / 2 * 2^e*
    (e is the least one that will do), so max_d sum_k p_k |v_kd| >= p* 2^e* Qmax / 2, and L keys give at most L 2^-29 of
    that maximum over d (it shows where an element's own sum leaves out the large rows)."""
    n, H, hd = q.shape
    KV, L = k.shape[1], k.shape[0]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    there = ~torch.isnan(k[:, 0, 0])
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    i, j = torch.arange(n)[:, None] + base, torch.arange(L)[None, :]
    ok = there[None, :].expand(n, L).clone()
    if not block:
        ok &= j <= i
        if window:
            ok &= i - j < window
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(H):
        kk, vv = k[:, h // (H // KV)], v[:, h // (H // KV)]
        s = q[:, h] @ kk.T * scale
        a = q[:, h].abs() @ kk.abs().T * abs(scale)
        s = torch.where(ok & torch.isfinite(s), s, torch.tensor(-math.inf, dtype=torch.float64))
        m = s.amax(-1, keepdim=True)
        p = torch.where(torch.isfinite(s), torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m))), torch.zeros_like(s))
        z = p.sum(-1, keepdim=True)
        p = torch.where(z > 0, p / z, torch.zeros_like(p))
        out[:, h] = p @ vv
        live = torch.where(torch.isfinite(s), a, torch.zeros_like(a)).amax(-1, keepdim=True)
        ds = live * (2.0 ** -22 + (hd + 8) * 2.0 ** -23) + 2.0 ** -22
        pv = p @ vv.abs()
        tol[:, h] = pv * (2 * ds + 2.0 ** -21 + (3 * L / 8 + 64) * 2.0 ** -23) + pv.amax(-1, keepdim=True) * L * 2.0 ** -29 + 1e-37
    return out, tol
