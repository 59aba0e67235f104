"""The quantised serving operators in 64 bits, from their definition, for the tests of them."""
from __future__ import annotations

import numpy as np

from irontensor_amd.tensor import bf16_to_f32, f32_to_bf16

TINY = 2.0 ** -126
GROUP = 32


def rne_bf16(x):
    return bf16_to_f32(f32_to_bf16(np.asarray(x, np.float32))).reshape(np.shape(x))


def steps(x, group, levels, bf16=True):
    """[.., D / group] FP32 steps of x [.., D]: max|x| * (1 / levels), NaN where a value is not finite."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // group, group)
    with np.errstate(invalid="ignore"):
        most = np.abs(g).max(-1)
        s = most * (np.float32(1) / np.float32(levels))
    if bf16:
        s = rne_bf16(s)
    s = np.where(s < TINY, np.float32(0), s)
    return np.where(np.isfinite(g).all(-1), s, np.float32(np.nan))


def codes(x, s, group, levels):
    """rne(x / s) in float64 (a quotient of two FP32 numbers of which one has at most 32 bits times a half
    is never mistaken there), 0 where the step is 0 or NaN."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // group, group)
    live = s > 0
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.rint(g / np.where(live, s, 1).astype(np.float64)[..., None])
    return np.where(live[..., None], np.clip(q, -levels, levels), 0).reshape(x.shape)


def stands_for(x, group, levels, bf16=True):
    s = steps(x, group, levels, bf16)
    return codes(x, s, group, levels) * np.repeat(s.astype(np.float64), group, -1)


def cache_values(k, v, bits):
    """What keys and values [.., D] read back as."""
    levels = 7 if bits == 4 else 127
    return stands_for(k, GROUP, levels), stands_for(v, v.shape[-1], levels)


def attend(q, k, v, start, count, scale):
    """q [B, n, H, D] over the values k, v [B, T, Hkv, D] in float64 -> (o, sum p|v|, largest scale * sum|q k| of a
    row, sum p max|v|, largest scale * sum over the groups of max|k| sum|q|); the last two for the offsets."""
    b, n, h, d = q.shape
    t, hkv = k.shape[1:3]
    o, pv, pm = (np.zeros(q.shape) for _ in range(3))
    mag, qm = np.zeros((b, n, h, 1)), np.zeros((b, n, h, 1))
    for bi in range(b):
        for i in range(min(n, max(0, int(count[bi])))):
            lim = min(max(int(start[bi]) + i + 1, 0), t)
            if lim == 0:
                continue
            for hi in range(h):
                kk, vv = k[bi, :lim, hi // (h // hkv)], v[bi, :lim, hi // (h // hkv)]
                x = q[bi, i, hi].astype(np.float64)
                s = kk @ x * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                o[bi, i, hi], pv[bi, i, hi] = p @ vv, p @ np.abs(vv)
                mag[bi, i, hi] = (np.abs(kk) @ np.abs(x)).max() * scale
                pm[bi, i, hi] = p @ np.abs(vv).max(-1)
                qm[bi, i, hi] = (np.abs(kk).reshape(lim, -1, GROUP).max(-1) @ np.abs(x).reshape(-1, GROUP).sum(-1)).max() * scale
    return o, pv, mag, pm, qm


def attend_bound(want, t, d, bf16):
    """Largest error of an element. FP32: a score is an FP32 sum of D products and D / 32 multiples of them, off by
    at most (D + 16) 2^-24 of the sum of their magnitudes; 2^x is off by 2^-21 for the sizes of x here, the
    scaled exponent's rounding among it (2^-24 |x|, |x| < 2^3 mag); a numerator and a denominator carry that,
    and sums of T terms, each off by at most T 2^-24. BF16: P rounded (2^-8 a term) and the output (2^-8); and
    its sums run on codes raised by up to 24 steps (4 bits: 16 + code + 8 <= 31 steps, max|x| = 7 steps; 8 bits:
    255 and 127), so that a sum's terms are up to 31 / 7 < 4.5 times the group's largest value, and their
    FP32 roundings, D 2^-24 in a score and T 2^-24 in an output, go by that."""
    o, pv, mag, pm, qm = want
    if bf16:
        mag = mag + 4.5 * qm
    e = 2 * ((d + 16 + 8) * 2.0 ** -24 * mag + 2.0 ** -21 + t * 2.0 ** -24) * pv
    if bf16:
        e = e + 2 * (t + 2) * 2.0 ** -24 * 4.5 * pm
    return e + (2.0 ** -8 * (pv + np.abs(o) + e) if bf16 else 2.0 ** -24 * np.abs(o))
