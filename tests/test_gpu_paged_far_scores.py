"""Paged attention over scores so large that 32 bits hold them in whole steps, in
every kernel."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import Dev, be, close, i32, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu

# routes: (H, Hkv, D, page size, lengths, query rows, groups, prefixes)
ROUTES = {
    "single rows": (8, 2, 64, 16, [4097, 300], None, None, None),
    "single rows, one by one": (4, 4, 128, 6, [4097, 300], None, None, None),
    "single rows of 16 heads": (16, 1, 128, 16, [4097, 300], None, None, None),
    "prefix": (8, 2, 64, 16, [4097, 4100, 4150], None, [0, 3], [4090]),
    "prefix of many rows": (16, 1, 128, 32, [4097] * 20, None, [0, 20], [4096]),
    "prompt": (2, 2, 128, 16, [4097, 300], [40, 7], None, None),
    "prompt that fills row blocks": (8, 2, 64, 16, [4097, 4200], [130, 100], None, None),
    "prompts behind a prefix": (4, 2, 128, 16, [4097, 4090, 4110], [12, 5, 20], [0, 3], [4064]),
}


@pytest.mark.parametrize("power", [10, 17, 19, 23, 26, 29, 33, 60])
@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_far_scores(be, s, dtype, cache, route, power):
    """Scores of 2^power and more, apart by as much: the largest takes the whole
    weight, so the result is its value, off by the weight's rounding, and that
    of the weights' sum, two products and a quotient."""
    H, Hkv, D, ps, lens, new, groups, prefix = ROUTES[route]
    rng = np.random.default_rng(power)
    B = len(lens)
    rows = -(-max(lens) // ps)
    table = np.arange(B * rows).reshape(B, rows)
    if prefix:
        for b in range(B):
            table[b, :prefix[0] // ps] = table[0, :prefix[0] // ps]
    ck = np.zeros((B * rows, ps, Hkv, D))
    ck[..., 0] = rng.uniform(-1, 1, ck.shape[:3])
    cv = rng.standard_normal((B * rows, ps, Hkv, D))
    for p in (0, 150):                                   # the larger one is seen by all or by none
        for b in range(B):
            ck[table[b, p // ps], p % ps, :, 0] = 2 + (p > 0)
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    T = B if new is None else int(starts[-1])
    q = np.zeros((T, H, D))
    q[..., 0] = rng.uniform(1, 2, (T, H))
    qd, kd, vd = Dev(be, q, dtype), Dev(be, ck, cache), Dev(be, cv, cache)
    tb, ln, o = i32(be, table), i32(be, lens), Dev(be, np.zeros((T, H, D)), dtype)
    opt = {n: (None if x is None else i32(be, x)) for n, x in
           (("query_starts", starts), ("group_starts", groups), ("prefix_lens", prefix))}
    be.paged_attention(s, qd.t, kd.t, vd.t, tb.t, ln.t, 2.0 ** power, out=o.t, **{n: x and x.t for n, x in opt.items()})
    s.synchronize()
    values, want = vd.f64(), np.zeros((T, H, D))
    for b in range(B):
        for j in range(1 if new is None else new[b]):
            seen = lens[b] if new is None else lens[b] - new[b] + j + 1
            p = 150 if seen > 150 else 0
            t = b if new is None else starts[b] + j
            want[t] = np.repeat(values[table[b, p // ps], p % ps], H // Hkv, 0)
    step = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    close(o.f64(), want, (step + 80 * 2.0 ** -23) * np.abs(want) + ref.rounding(want, dtype))
