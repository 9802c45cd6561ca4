"""Paged attention whose CTAs hold long stretches of one row tile: with 32-bit
queries such a stretch is done in pieces whose sums are joined with rounding."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import Dev, be, check_attention, close, i32, make_cache, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu

# More than 10 key tiles of 128 of a row tile for a CTA (of 148, one row tile at
# a time): H, Hkv, D, page size, lengths, query rows, groups, prefixes
SHAPES = {
    # 24 x 8 row tiles of 11 to 15 key tiles, 17 a CTA: some whole, some cut
    "prompts": (8, 8, 64, 16, [1300 + 26 * i for i in range(24)], [5 - i % 3 for i in range(24)], None, None),
    "prompts, one by one": (8, 8, 64, 12, [1300 + 26 * i for i in range(24)], [5 - i % 3 for i in range(24)], None, None),
    # 12 x 8 of 24: all cut
    "long prompts": (16, 8, 128, 32, [3000 - 7 * i for i in range(12)], [3] * 12, None, None),
    # 12 groups x 8 of 20 tiles; one sequence of each holds less than the prefix, one nothing
    "prefixes": (8, 8, 64, 16, [2600, 2510, 100, 0] * 12, None, list(range(0, 49, 4)), [2500] * 12),
    "prompts behind prefixes": (8, 8, 64, 16, [2600, 2530, 100] * 12, [4, 30, 7] * 12, list(range(0, 37, 3)), [2500] * 12),
    # row blocks that fill a tile, their prefix ends inside a page
    "prompts that fill row tiles": (4, 4, 64, 16, [1500 + 9 * i for i in range(18)], [129, 64, 200] * 6, list(range(0, 19, 3)), [1205] * 6),
}


def inputs(be, name, dtype, cache):
    H, Hkv, D, ps, lens, new, groups, prefix = SHAPES[name]
    rng = np.random.default_rng(len(name))
    ck, cv, table = make_cache(be, rng, -(-max(lens) // ps), lens, ps, Hkv, D, cache, groups, prefix)
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    T = len(lens) if new is None else int(starts[-1])
    return rng, Dev(be, rng.standard_normal((T, H, D)) * 2, dtype), ck, cv, table, lens, starts, groups, prefix


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_long_stretches(be, s, dtype, cache, name):
    rng, q, ck, cv, table, lens, starts, groups, prefix = inputs(be, name, dtype, cache)
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache, starts, groups, prefix)


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_sums_of_32_bit_queries(be, s, name):
    """Equal scores: means of values between 1 and 2. The matrix unit cuts its
    sum after each product of 16 keys, by up to 2^-23 of it: 5 tiles of a stream
    in two parts, 80 products, between two joins with rounding (three operations
    each, at most 24 pieces and 24 CTAs)."""
    rng, q, ck, cv, table, lens, starts, groups, prefix = inputs(be, name, "f32", "f16")
    q.x.zero_()
    cv.x.copy_((cv.x.abs() % 1.0) + 1.0)
    opt = {n: (None if x is None else i32(be, x)) for n, x in
           (("query_starts", starts), ("group_starts", groups), ("prefix_lens", prefix))}
    o, tb, ln = Dev(be, np.zeros(tuple(q.x.shape))), i32(be, table), i32(be, lens)
    be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 1.0, out=o.t, **{n: x and x.t for n, x in opt.items()})
    s.synchronize()
    want, _ = ref.attention(q.f64(), np.nan_to_num(ck.f64()), cv.f64(), table, lens, 1.0, starts, groups, prefix)
    close(o.f64(), want, (80 + 3 * 48 / 2 + 8) * 2.0 ** -23 * np.abs(want))
