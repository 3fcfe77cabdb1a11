"""Rows held in 4 bits, in 64 bits on the CPU: what a cache of given rows holds, and
what given bytes stand for."""
import numpy as np
import torch

import _cachetight as tight

CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
TABLE = np.concatenate((CODES, -CODES))


def step_type(dt):
    return torch.float16 if dt == torch.float16 else torch.bfloat16


def steps(x):
    """Steps (..., ng) in 64 bits of rows x (..., D): the largest magnitude of 64
    elements over 6, to 6 significant bits, ties to even. NaN where a group is not finite."""
    half = x.dtype == torch.float16
    a = x.detach().cpu().double().abs().numpy()
    ng = -(-a.shape[-1] // 64)
    out = np.empty((*a.shape[:-1], ng))
    for g in range(ng):
        with np.errstate(invalid="ignore"):
            want = a[..., 64 * g:64 * g + 64].max(-1) / 6
            unit = np.ldexp(1.0, np.maximum(np.frexp(want)[1] - 6, -23 if half else -125))
            s = np.minimum(np.rint(want / unit) * unit, 10752.0 if half else 42 * 2.0 ** 120)
        out[..., g] = np.where(np.isfinite(want), s, np.nan)
    return out


def held(k, v):
    """The values that a cache holds for rows k, v (..., D): each x / step to the nearest
    code, the even one of two as near, by looking at all of them."""
    sk, sv = steps(k), steps(v)
    bad = np.isnan(sk).any(-1, keepdims=True) | np.isnan(sv).any(-1, keepdims=True)
    out = []
    for x, s in ((k, sk), (v, sv)):
        s = np.repeat(np.where(bad, np.nan, s), 64, axis=-1)[..., :x.shape[-1]]
        y = x.detach().cpu().double().numpy()
        with np.errstate(invalid="ignore"):
            off = np.abs(np.abs(y)[..., None] - CODES * s[..., None])
            off = np.where(np.isnan(off), 0.0, off)
            near = off == off.min(-1, keepdims=True)
            even = near & (np.arange(8) % 2 == 0)
            pick = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
            out.append(torch.from_numpy(np.where(y < 0, -1.0, 1.0) * CODES[pick] * s))
    return out


def decode(codes, step):
    """What bytes (..., D / 2) and steps (..., ng) stand for, in 64 bits."""
    c, s = codes.cpu().numpy(), step.detach().cpu().double().numpy()
    x = np.empty((*c.shape[:-1], 2 * c.shape[-1]))
    x[..., 0::2], x[..., 1::2] = TABLE[c & 15], TABLE[c >> 4]
    return torch.from_numpy(x * np.repeat(s, 64, axis=-1)[..., :x.shape[-1]])


def values(held):
    """Key and value rows of (k4, v4, step), in 64 bits."""
    k4, v4, step = held
    return decode(k4, step[..., 0, :]), decode(v4, step[..., 1, :])


def check_attend(got, held, q, lens, count=None, scale=None, gate=None):
    """Attention over a cache against the formula over its values (the bounds of
    _cachetight). The products are exact: a 32-bit query goes as three bf16 numbers,
    of which the second and third are at most 2^-7 and 2^-14 of the first, so the
    roundings of their sums are those of at most D (1 + 2^-7 + 2^-14) <= D + 3 terms of
    the score's absolute sum; joining the pieces is two more and applying up to 4
    groups' steps and adding them up at most 8. So 13 steps more than the D + 4 of the
    bounds, whose `big` is scaled by them, and P's product with a value's step, one more
    rounding of each p, is covered by the 2^-20 = 16 steps that they hold for p itself.
    Numbers below 2^-126 count as zero in the exponential and in the products: each p
    (at most 1, the row's sum at least 1) may lose 2^-126 there, its product with the step
    the same twice (steps here are above 2^-4, so at most 2^-122 of v), and each piece of
    that as much, three of them: less than 2^-120 of sum |v| in all. Added to the `a`
    of the bounds, which counts 2 * 2^-20 of it or more, as 2^-101 of sum |v|.
    fp16 results below 2^-14 are multiples of 2^-24, off by up to 2^-25 whatever their size:
    the bounds have that for an element but not for the L2 error, whose square it makes
    2^-50 / 3 larger for each element. They take h^2 / 3 = 2^-22 / 3 of sum p^2 v^2, to
    which 2^-28 is added. (6144 such results: sqrt(6144 / 3) 2^-25 = 1.35e-6.)"""
    k, v = values(held)
    r = tight.attend(q, k, v, lens, count, None, None, scale, gate, None)
    D = q.shape[-1]
    r["big"] *= (D + 17) / (D + 4)
    r["a"] = r["a"] + 2.0 ** -101 * r["v1"]
    if q.dtype == torch.float16:
        r["a2"] = r["a2"] + 2.0 ** -28
    rounded = q.shape[2] * (q.shape[1] // k.shape[1]) > 16
    tight.check((*got, None), r, q, k.shape[2], rounded and q.dtype != torch.float32, gate is not None)
