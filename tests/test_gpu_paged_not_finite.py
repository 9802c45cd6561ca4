"""Paged attention over queries and keys that are not finite."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import PAIRS, Dev, be, close, i32, make_cache, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu

# (H, Hkv, D, page size, lengths, query rows, groups, prefixes); the second
# sequence's keys lie in several parts of the line, the third's in one
ROUTES = {
    "single rows": (8, 2, 64, 16, [40, 3000, 64], None, None, None),
    "single rows, one by one": (8, 2, 64, 6, [40, 3000, 64], None, None, None),
    "prefix": (8, 2, 64, 16, [640, 3000, 650], None, [0, 3], [600]),
    "prompts": (8, 2, 128, 16, [40, 3000, 64], [5, 40, 9], None, None),
    "prompts that fill row blocks": (8, 2, 64, 16, [150, 900, 180], [100, 100, 120], None, None),
    "prompts behind a prefix": (4, 2, 64, 16, [640, 3000, 650], [5, 9, 3], [0, 3], [600]),
}


class Case:
    def __init__(self, be, dtype, cache, route):
        self.be, self.dtype, self.cache = be, dtype, cache
        self.H, self.Hkv, self.D, self.ps, self.lens, self.new, self.groups, self.prefix = ROUTES[route]
        rng = np.random.default_rng(41)
        B = len(self.lens)
        self.ck, self.cv, self.table = make_cache(be, rng, -(-max(self.lens) // self.ps), self.lens, self.ps, self.Hkv, self.D,
                                                  cache, self.groups, self.prefix)
        self.starts = np.arange(B + 1) if self.new is None else np.concatenate([[0], np.cumsum(self.new)])
        self.q = Dev(be, rng.standard_normal((self.starts[-1], self.H, self.D)), dtype)

    def key(self, b, p):
        """Where position p of sequence b lies, as the attention reads it."""
        first = self.groups[0] if self.prefix and p < self.prefix[0] else b
        return int(self.table[first][p // self.ps]), p % self.ps

    def run(self, s):
        opt = {n: (None if x is None else i32(self.be, x)) for n, x in
               (("query_starts", None if self.new is None else self.starts), ("group_starts", self.groups), ("prefix_lens", self.prefix))}
        o, tb, ln = Dev(self.be, np.zeros(tuple(self.q.x.shape)), self.dtype), i32(self.be, self.table), i32(self.be, self.lens)
        self.scale = float(np.float32(self.D ** -0.5))
        self.be.paged_attention(s, self.q.t, self.ck.t, self.cv.t, tb.t, ln.t, self.scale, out=o.t,
                                **{n: x and x.t for n, x in opt.items()})
        s.synchronize()
        return o.f64()

    def check(self, s, q=None, ck=None, nan=()):
        """Against the definition (with q and ck in place of the tensors'), rows `nan` all NaN."""
        got = self.run(s)
        with np.errstate(invalid="ignore"):
            q, ck = self.q.f64() if q is None else q, self.ck.f64() if ck is None else ck
            rest = self.cv.f64(), self.table, self.lens, self.scale, self.starts, self.groups, self.prefix
            want, _ = ref.attention(q, ck, *rest)
            _, info = ref.attention(q, np.where(np.isinf(ck), 0.0, ck), *rest)   # sizes of the finite scores
        there = np.ones(len(want), bool)
        there[list(nan)] = False
        assert np.isnan(got[~there]).all(), f"{(~np.isnan(got[~there])).sum()} values of {got[~there].size} are numbers"
        close(got[there], want[there], ref.attention_bound(want[there], info[there], self.dtype, self.cache, self.D))


@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_a_query_that_is_no_number(be, s, dtype, cache, route):
    for b in range(3):
        c = Case(be, dtype, cache, route)
        row = int(c.starts[b])
        clean = c.q.f64()
        c.q.x[row, :, 3] = float("nan")
        c.check(s, q=clean, nan=[row])


@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("at", ["first", "next", "last"])
def test_a_key_that_is_no_number(be, s, dtype, cache, route, at):
    """NaN wherever it stands among the keys that a query sees."""
    c = Case(be, dtype, cache, route)
    b = 1
    p = {"first": 0, "next": 5, "last": c.lens[b] - 1}[at]
    clean = c.ck.f64()
    page, r = c.key(b, p)
    c.ck.x[page, r, :, 7] = float("nan")
    rows = []
    for k in range(3):
        n = c.starts[k + 1] - c.starts[k]
        for j in range(n):
            if p <= c.lens[k] - n + j and c.key(k, p) == (page, r):
                rows.append(c.starts[k] + j)
    assert rows
    c.check(s, ck=clean, nan=rows)


@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", [p for p in PAIRS if p != ("f32", "f16")])
def test_scores_of_minus_infinity(be, s, dtype, cache, route):
    """A score of -inf takes no weight; a query that has no others gives zeros."""
    c = Case(be, dtype, cache, route)
    c.q.x[..., 0] = 1.0
    c.ck.x[..., 0] = float("-inf")
    assert not c.run(s).any()
    c = Case(be, dtype, cache, route)
    c.q.x[..., 0] = 1.0
    for b in range(3):
        for p in range(0, c.lens[b] - (c.new[b] if c.new else 0), 3):
            page, r = c.key(b, p)
            c.ck.x[page, r, :, 0] = float("-inf")
    c.check(s)


@pytest.mark.parametrize("route", sorted(ROUTES))
@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_a_score_of_infinity(be, s, dtype, cache, route):
    """inf - inf: no number, like the definition's; other sequences hold."""
    c = Case(be, dtype, cache, route)
    c.q.x[..., 0] = 1.0
    clean = c.ck.f64()
    p = c.lens[2] - 1
    page, r = c.key(2, p)
    c.ck.x[page, r, :, 0] = float("inf")
    c.check(s, ck=clean, nan=[int(c.starts[3]) - 1])
