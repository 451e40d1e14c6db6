"""How far attention over the paged cache is off on average: a bound that one lost plane of Q or P, or tensor-core sums that
are never folded, pass by far (the worst-case bound of paged_ref grows with the length and the head and does not see them)."""
from __future__ import annotations

import math

import torch


def steps(chunk: bool, hd: int, L: int):
    """(products summed for a score, products summed for an output before they are folded): 16-deep, and the chunk kernel
    puts both planes into one sum."""
    fold = 512 if chunk else 256
    planes = 2 if chunk else 1
    return planes * hd // 16, planes * min(fold, L) // 16


def rms_bound(chunk: bool, hd: int, L: int, s: float) -> float:
    """Bound of rms(error) / rms(output) for values of V that are independent, symmetric and of one size; s: rms of the
    scores (before the maximum is subtracted; scores within 8 of each other count).

    An output is sum_k p_k v_k, its error sum_k p_k eps_k v_k with the relative errors eps_k of the weights, which know
    nothing of V: over V the expected squares are sum p_k^2 and sum p_k^2 eps_k^2, so the ratio of their roots is at most
    max |eps_k|, or its rms where eps varies. The errors of a weight, each with its largest relative size:
      q in two planes              2^-22 s                 (22 bits; the terms of a score have random signs)
      tensor-core sums of a score  n 2^-23 s               (n sums cut below 24 bits; partial sums are at most s on average)
      scale, maximum, 2^x          4 * 2^-24 * 8 + 2^-22   (four roundings of numbers up to 8 log2 e in the exponent, x ln 2)
      p in two planes              2^-22
    and of the output: the tensor cores' cut, n' 2^-23 of partial sums that are at most what is folded then; the folds,
    the sum of the weights, the merge of warps or pieces and the division 2^-21."""
    n, npv = steps(chunk, hd, L)
    return (2.0 ** -22 + n * 2.0 ** -23) * s + 32 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -22 + npv * 2.0 ** -23 + 2.0 ** -21


def pull_bound(chunk: bool, hd: int, L: int) -> float:
    """Bound of the mean signed relative error for values of V of one sign: partial sums grow evenly, so a cut of at most
    2^-23 takes half of that on average, 2^-24 for each product between two folds; what is left has no preferred sign
    and the sums of weights round, 2^-21 for all of it."""
    return steps(chunk, hd, L)[1] * 2.0 ** -24 + 2.0 ** -21


def exact(q, k, v, base, scale, dtype=torch.float64):
    """q [n, H, hd], k / v [L, KV, hd], causal: (out [n, H, hd], rms score); float64 on whatever device q is on."""
    n, H, hd = q.shape
    L, KV = k.shape[:2]
    q, k, v = (x.to(dtype) for x in (q, k, v))
    s = torch.einsum("ikgd,jkd->kgij", q.view(n, KV, H // KV, hd), k) * scale
    seen = torch.arange(L, device=q.device)[None, :] <= base + torch.arange(n, device=q.device)[:, None]
    size = math.sqrt(float((s * seen).square().sum() / (seen.sum() * H)))
    p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    return torch.einsum("kgij,jkd->ikgd", p, v).reshape(n, H, hd), size


def ratio(got, want) -> float:
    return math.sqrt(float((got.double() - want).square().mean() / want.square().mean()))


def pull(got, want) -> float:
    return float(((got.double() - want) / want).mean())
