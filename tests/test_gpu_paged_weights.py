"""Paged attention whose small weights matter: one key far above thousands of
equal ones (an attention sink), in every kernel."""
import math

import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import Dev, be, close, i32, s  # noqa: F401 (be, s: fixtures)
from test_gpu_paged_far_scores import ROUTES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [10.0, 12.0, 17.0, 18.0])
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_small_weights_beside_a_large_one(be, s, dtype, cache, route, at, gap):
    """One key has the score `gap` and the value 0, the others 0 and 1: a query
    that sees n others gives n w / (1 + n w), w = e^-gap.

    The scores are single products of exact values, so the weights are off by
    the rounding of scale log2(e) and of the score (2^-23 of gap log2(e) in the
    exponent, ln 2 of that relative), 2^-22 for each of two exponentials, and by
    their own rounding for the value product: half a step of their type, or
    2^-22 in two parts, and never more than 2^-36 of the largest. Value and
    weight sums of n terms as in attention_bound."""
    H, Hkv, D, ps, lens, new, groups, prefix = ROUTES[route]
    B = len(lens)
    rows = -(-max(lens) // ps)
    table = np.arange(B * rows).reshape(B, rows)
    if prefix:
        for b in range(B):
            table[b, :prefix[0] // ps] = table[0, :prefix[0] // ps]
    ck, cv = np.zeros((B * rows, ps, Hkv, D)), np.ones((B * rows, ps, Hkv, D))
    sink = []
    for b in range(B):
        seen = lens[b] if new is None else lens[b] - new[b] + 1      # what its first query sees
        p = {"first": 0, "middle": seen // 2, "last": seen - 1}[at]
        if prefix and at != "first":
            p = min(p, prefix[0] - 1) if at == "middle" else p
            p = sink[0] if at == "middle" and b else p                # one key for the group
        sink.append(p)
        t = 0 if prefix and p < prefix[0] else b                      # the prefix is read through the first
        ck[table[t, p // ps], p % ps, :, 0] = gap / 4
        cv[table[t, p // ps], p % ps] = 0
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    T = B if new is None else int(starts[-1])
    q = np.zeros((T, H, D))
    q[..., 0] = 4
    qd, kd, vd = Dev(be, q, dtype), Dev(be, ck, cache), Dev(be, cv, cache)
    tb, ln, o = i32(be, table), i32(be, lens), Dev(be, np.zeros((T, H, D)), dtype)
    opt = {n: (None if x is None else i32(be, x)) for n, x in
           (("query_starts", starts), ("group_starts", groups), ("prefix_lens", prefix))}
    be.paged_attention(s, qd.t, kd.t, vd.t, tb.t, ln.t, 1.0, out=o.t, **{n: x and x.t for n, x in opt.items()})
    s.synchronize()
    w = math.exp(-gap)
    n = np.zeros(T)
    for b in range(B):
        for j in range(1 if new is None else new[b]):
            n[b if new is None else starts[b] + j] = (lens[b] if new is None else lens[b] - new[b] + j + 1)
    n = n[:, None, None] - 1                                          # every query sees the large one
    want = np.broadcast_to(n * w / (1 + n * w), (T, H, D))
    step = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    rel = max(step, 2.0 ** -36 / w) + gap * 2.0 ** -23 + 2 * 2.0 ** -22 + (n / 8 + 64) * 2.0 ** -23
    close(o.f64(), want, rel * want + ref.rounding(want, dtype), f"gap {gap}")
