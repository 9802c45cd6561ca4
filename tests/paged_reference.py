"""The rotary, head-norm, paged-append and paged-attention operations from
their definitions in 64 bits, one loop per row, and the error bounds of the
device's arithmetic (half a step per rounding, counted)."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# f16 values below 2^-14 stand 2^-24 apart, so rounding to one moves by up to
# 2^-25 whatever the value is
HALF_TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
U32 = 2.0 ** -24


def rounding(y, dtype):
    return HALF_STEP[dtype] * np.abs(y) + HALF_TINY[dtype]


def frequencies(theta, d, scaling="none", factor=1.0, orig=0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0,
                freq_factors=None):
    out = []
    for i in range(d // 2):
        f = theta ** (-2.0 * i / d)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            lo, hi = (d * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (beta_fast, beta_slow))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - r) + f / factor * r
        elif scaling == "bands":
            m = min(1.0, max(0.0, (orig * f / (2 * math.pi) - low) / (high - low)))
            f = m * f + (1 - m) * f / factor
        out.append(f / (1.0 if freq_factors is None else float(freq_factors[i])))
    return np.array(out)


def amplitude(scaling, factor):
    return 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


def rotate(x, positions, freq, half_layout, amp=1.0):
    """x [T, H, D] f64; the first 2 len(freq) values turn."""
    y, d = x.copy(), 2 * len(freq)
    ang = np.asarray(positions, dtype=np.float64)[:, None, None] * freq
    c, s = np.cos(ang) * amp, np.sin(ang) * amp
    a, b = (np.s_[..., :d // 2], np.s_[..., d // 2:d]) if half_layout else (np.s_[..., 0:d:2], np.s_[..., 1:d:2])
    y[a] = x[a] * c - x[b] * s
    y[b] = x[a] * s + x[b] * c
    return y


def rms(x, w, eps):
    return x * w / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def rotate_bound(x, y, dtype, amp=1.0):
    """cos and sin are off by pi 2^-24 (the turn rounded to 32 bits) and 2 units
    of 2^-23 (sincospi's and the amplitude's rounding); a value is u c - w s:
    two such errors, two products and a sum, then the output's rounding."""
    return (2 * (math.pi + 4) + 3) * U32 * amp * np.abs(x).max(-1, keepdims=True) + rounding(y, dtype)


def attention(q, ck, cv, table, lens, scale, starts=None, group_starts=None, prefix_lens=None):
    """out f64 (rows of no sequence are NaN), and per row (S, n, vmax): the
    largest sum of |q k| scale, the keys seen and the largest |value|."""
    T, H, D = q.shape
    Hkv, ps = ck.shape[2], ck.shape[1]
    g = H // Hkv
    out = np.full(q.shape, np.nan)
    info = np.zeros((T, 3))
    B = len(lens)
    starts = np.arange(B + 1) if starts is None else starts
    for b in range(B):
        n = starts[b + 1] - starts[b]
        prefix, first = 0, b
        if group_starts is not None:
            for k in range(len(prefix_lens)):
                if group_starts[k] <= b < group_starts[k + 1]:
                    prefix, first = int(prefix_lens[k]), int(group_starts[k])
        rows = [(table[first if p < prefix else b][p // ps], p % ps) for p in range(int(lens[b]))]
        at = np.array(rows, dtype=np.int64).reshape(-1, 2)
        K, V = ck[at[:, 0], at[:, 1]], cv[at[:, 0], at[:, 1]]
        for j in range(n):
            t = starts[b] + j
            see = max(0, int(lens[b]) - n + j + 1)
            out[t] = 0.0
            if see == 0:
                continue
            for h in range(Hkv):
                k, v, x = K[:see, h], V[:see, h], q[t, h * g:(h + 1) * g]
                s = x @ k.T * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                out[t, h * g:(h + 1) * g] = (p / p.sum(-1, keepdims=True)) @ v
                info[t, 0] = max(info[t, 0], (np.abs(x) @ np.abs(k).T).max() * abs(scale))
            info[t, 1], info[t, 2] = see, np.abs(V[:see]).max()
    return out, info


def attention_bound(out, info, dtype, cache, D):
    """Scores: a sum of D products in 32 bits in any order, the query in parts
    that leave 2^-22 of it: (D + 4 + 4) 2^-24 S. Weights: twice that, 2^-22 for
    the exponential, and their rounding for the value product (to the cache's
    type, or in two parts when the result has 32 bits: 2^-22). Values: a sum of
    n terms in 32 bits that may truncate (2^-23 per 8 terms, and 64 joins of
    parts); then the output's rounding."""
    S, n, v = (info[:, i][:, None, None] for i in range(3))
    weight = 2.0 ** -22 if dtype == "f32" else HALF_STEP[cache]
    rel = 2 * (D + 8) * U32 * S + 2.0 ** -22 + weight + (n / 8 + 64) * 2.0 ** -23
    return rel * v + rounding(out, dtype) + 1e-30
