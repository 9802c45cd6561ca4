"""Rotary forms, head norms, cache append and attention over paged caches, on
the device against their definitions in 64 bits (paged_reference.py)."""
import ctypes
import math

import numpy as np
import pytest

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_():
    import torch
    return torch


@pytest.fixture(scope="module")
def be(cuda_lib):
    from beacon_cuda import CudaBackend
    return CudaBackend(0)


@pytest.fixture(scope="module")
def s(be):
    return be.new_stream()


class Dev:
    """A torch tensor and the framework's view of it, `offset` values into its storage."""

    def __init__(self, be, x, dtype=None, offset=0):
        import torch
        from beacon_cuda import _lib as L
        dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}[dtype or "f32"]
        kind = {"f32": L.DTYPE_F32, "f16": L.DTYPE_F16, "bf16": L.DTYPE_BF16, "i32": L.DTYPE_I32}[dtype or "f32"]
        x = torch.as_tensor(np.asarray(x)).to(dt)
        store = torch.empty(x.numel() + offset + 8, dtype=dt, device="cuda")
        self.x = store[offset:offset + x.numel()].view(x.shape)
        self.x.copy_(x)
        torch.cuda.synchronize()
        self.t = be.wrap(self.x.data_ptr(), tuple(x.shape), kind)

    def f64(self):
        return self.x.double().cpu().numpy()


def i32(be, v):
    return Dev(be, np.asarray(v, dtype=np.int32), "i32")


def close(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / bound):.3g} of the bound"


SCALINGS = {"none": {}, "linear": dict(factor=4.0), "yarn": dict(factor=8.0, orig=2048),
            "bands": dict(factor=8.0, orig=4096)}


def make_rope(be, theta, rd, layout, scaling, **more):
    from beacon_cuda import _lib as L
    p = SCALINGS[scaling]
    kind = {"none": L.ROPE_SCALING_NONE, "linear": L.ROPE_SCALING_LINEAR, "yarn": L.ROPE_SCALING_YARN,
            "bands": L.ROPE_SCALING_BANDS}[scaling]
    h = be.rope_create(theta, rd, L.ROPE_HALF if layout == "half" else L.ROPE_INTERLEAVED, kind, p.get("factor", 1.0),
                       p.get("orig", 0), **more)
    return h, ref.frequencies(theta, rd, scaling, **p, **more), ref.amplitude(scaling, p.get("factor", 1.0))


# --- rotary forms ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("scaling", sorted(SCALINGS))
@pytest.mark.parametrize("T,H,D,rd", [(1, 32, 128, 128), (7, 3, 128, 96), (33, 1, 64, 16)])
def test_rope_scaled(be, s, dtype, layout, scaling, T, H, D, rd):
    rng = np.random.default_rng(T * 100 + D)
    x = Dev(be, rng.standard_normal((T, H, D)) * 3, dtype)
    pos = rng.integers(0, 200000, T)
    rope, freq, amp = make_rope(be, 500000.0, rd, layout, scaling)
    out = be.rope_scaled(s, x.t, i32(be, pos).t, rope, out=None)
    o = Dev(be, np.zeros((T, H, D)), dtype)
    p = i32(be, pos)
    be.rope_scaled(s, x.t, p.t, rope, out=o.t)
    s.synchronize()
    want = ref.rotate(x.f64(), pos, freq, layout == "half", amp)
    close(o.f64(), want, ref.rotate_bound(x.f64(), want, dtype, amp))
    assert out.shape == (T, H, D) and out.dtype == x.t.dtype
    assert np.array_equal(out.read_raw(x.x.numel() * x.x.element_size()), o.t.read_raw(x.x.numel() * x.x.element_size()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("T,H,D,rd,offset", [(3, 2, 6, 4, 0), (2, 5, 80, 20, 0), (4, 3, 128, 128, 1), (2, 2, 7, 2, 3),
                                             (1, 1, 512, 512, 0), (2, 1, 512, 384, 0), (5, 70, 64, 64, 0),
                                             (300, 2, 96, 48, 0), (9, 3, 24, 12, 0), (700, 3, 64, 20, 0)])
def test_rope_odd_sizes_and_alignment(be, s, dtype, layout, T, H, D, rd, offset):
    """Head sizes and addresses that 16-byte loads do not fit, and the largest head."""
    rng = np.random.default_rng(D + offset)
    x = Dev(be, rng.standard_normal((T, H, D)), dtype, offset)
    pos = rng.integers(-5, 1 << 20, T)
    rope, freq, amp = make_rope(be, 10000.0, rd, layout, "none")
    p = i32(be, pos)
    want = ref.rotate(x.f64(), pos, freq, layout == "half")
    bound = ref.rotate_bound(x.f64(), want, dtype)
    be.rope_scaled(s, x.t, p.t, rope, out=x.t)   # in place
    s.synchronize()
    close(x.f64(), want, bound)


def test_rope_matches_the_unscaled_op(be, s):
    """rope_scaled at consecutive positions is op_rope in token-major order."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 4, 9, 64)).astype(np.float32)
    a = be.rope(s, be.upload(x), 37, 10000.0, 64).numpy()
    xt = Dev(be, np.ascontiguousarray(x[0].transpose(1, 0, 2)))
    rope, _, _ = make_rope(be, 10000.0, 64, "interleaved", "none")
    p = i32(be, 37 + np.arange(9))
    b = be.rope_scaled(s, xt.t, p.t, rope).numpy().transpose(1, 0, 2)
    # op_rope's angle is a 32-bit product of a 32-bit power: 46 * 4 * 2^-24 off at worst
    assert np.abs(a[0] - b).max() <= (46 * 4 + 24) * 2.0 ** -24 * 2 * np.abs(x).max()


def test_rope_frequency_factors(be, s):
    rng = np.random.default_rng(6)
    ff = rng.uniform(1, 8, 32).astype(np.float32)
    rope, freq, amp = make_rope(be, 10000.0, 64, "half", "linear", freq_factors=ff)
    x, p = Dev(be, rng.standard_normal((5, 2, 64))), i32(be, [0, 1, 77, 4096, 100000])
    o = be.rope_scaled(s, x.t, p.t, rope).numpy()
    want = ref.rotate(x.f64(), [0, 1, 77, 4096, 100000], freq, True)
    close(o, want, ref.rotate_bound(x.f64(), want, "f32"))


def test_rope_no_rows(be, s):
    rope, _, _ = make_rope(be, 10000.0, 64, "half", "none")
    o = be.rope_scaled(s, be.zeros((0, 4, 64)), be.zeros((0,), 3), rope)
    s.synchronize()
    assert o.shape == (0, 4, 64)


# --- norms of queries and keys ------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("T,H,Hkv,D,rd,wdtype", [(1, 32, 8, 128, 128, "f32"), (5, 4, 1, 64, 32, "f16"), (40, 6, 6, 96, 96, "f32"),
                                                 (3, 2, 1, 20, 12, "f16"), (2, 1, 1, 512, 512, "f32")])
def test_qk_norm_rope(be, s, dtype, layout, T, H, Hkv, D, rd, wdtype):
    rng = np.random.default_rng(D + T)
    q, k = Dev(be, rng.standard_normal((T, H, D)) * 2, dtype), Dev(be, rng.standard_normal((T, Hkv, D)) * 0.1, dtype)
    qw, kw = Dev(be, 1 + 0.3 * rng.standard_normal(D), wdtype), Dev(be, 1 + 0.3 * rng.standard_normal(D), wdtype)
    pos = rng.integers(0, 100000, T)
    rope, freq, amp = make_rope(be, 1e6, rd, layout, "bands")
    p, eps = i32(be, pos), 1e-6
    oq, ok = Dev(be, np.zeros((T, H, D)), dtype), Dev(be, np.zeros((T, Hkv, D)), dtype)
    be.qk_norm_rope(s, q.t, k.t, qw.t, kw.t, eps, p.t, rope, out_q=oq.t, out_k=ok.t)
    nq, nk = be.qk_norm_rope(s, q.t, k.t, qw.t, kw.t, eps)   # the norm alone
    s.synchronize()
    for x, w, o, n in ((q, qw, oq, nq), (k, kw, ok, nk)):
        y = ref.rms(x.f64(), w.f64(), float(np.float32(eps)))
        want = ref.rotate(y, pos, freq, layout == "half", amp)
        # the mean of squares: one rounding a value and one a join, half of it
        # after the root; root, quotient and two products
        norm = (D / 2 + 8) * 2.0 ** -24
        close(o.f64(), want, ref.rotate_bound(y, want, dtype, amp) + 2 * norm * np.abs(y).max(-1, keepdims=True))
        kind = {"f32": np.float32, "f16": np.float16}.get(dtype)
        if kind:
            close(n.numpy().astype(np.float64), y, norm * np.abs(y) + ref.rounding(y, dtype))
    be.qk_norm_rope(s, q.t, k.t, qw.t, kw.t, eps, p.t, rope, out_q=q.t, out_k=k.t)   # in place
    s.synchronize()
    assert np.array_equal(q.f64(), oq.f64()) and np.array_equal(k.f64(), ok.f64())


def test_qk_norm_of_zeros(be, s):
    z, w = Dev(be, np.zeros((2, 3, 64))), Dev(be, np.ones(64))
    oq, ok = be.qk_norm_rope(s, z.t, z.t, w.t, w.t, 1e-5)
    assert not oq.numpy().any() and not ok.numpy().any()


# --- cache append ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                         ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("ps,Hkv,D,rd,layout", [(16, 8, 128, 128, "interleaved"), (1, 1, 64, 32, "half"), (24, 3, 80, 0, "half"),
                                                (5, 2, 12, 6, "half")])
def test_paged_append(be, s, dtype, cache, ps, Hkv, D, rd, layout):
    rng = np.random.default_rng(ps * 7 + D)
    B, MP = 5, 9
    pages = B * MP + 3
    table = rng.permutation(pages)[:B * MP].reshape(B, MP)
    new = [1, 4, 0, 7, 2]
    held = rng.integers(0, MP * ps - 7 + 1, B) if ps > 1 else np.array([0, 5, 8, 2, 7])
    ids = np.repeat(np.arange(B), new)
    pos = np.concatenate([h + np.arange(n) for h, n in zip(held, new)])
    order = rng.permutation(len(ids))
    ids, pos = ids[order], pos[order]
    pos[3] = -1                                        # padding
    T = len(ids)
    k, v = Dev(be, rng.standard_normal((T, Hkv, D)), dtype), Dev(be, rng.standard_normal((T, Hkv, D)), dtype)
    ck, cv = (Dev(be, rng.standard_normal((pages, ps, Hkv, D)), cache) for _ in range(2))
    wk, wv = ck.f64(), cv.f64()
    rope, freq, amp = make_rope(be, 10000.0, rd, layout, "yarn") if rd else (None, np.zeros(0), 1.0)
    turned = ref.rotate(k.f64(), pos, freq, layout == "half", amp)
    bk, bv = np.zeros_like(wk), np.zeros_like(wv)
    edge = ref.rotate_bound(k.f64(), turned, cache, amp)
    for t in range(T):
        if pos[t] >= 0:
            at = table[ids[t]][pos[t] // ps], pos[t] % ps
            wk[at], wv[at], bk[at] = turned[t], v.f64()[t], edge[t]
            bv[at] = ref.rounding(wv[at], cache)
    tb, i, p = i32(be, table), i32(be, ids), i32(be, pos)
    be.paged_append(s, ck.t, cv.t, k.t, v.t, tb.t, p.t, seq_ids=i.t, rope=rope)
    s.synchronize()
    close(ck.f64(), wk, bk, "keys")
    close(cv.f64(), wv, bv, "values")


def test_paged_append_one_row_per_sequence_and_bad_indices(be, s):
    from beacon_cuda import ShapeMismatch
    rng = np.random.default_rng(3)
    B, ps, Hkv, D = 6, 4, 2, 64
    table = np.arange(B * 2).reshape(B, 2)
    table[2, 1] = 99                                   # no such page
    table[3, 0] = -1
    pos = np.array([0, 7, 4, 1, 8, 3])                 # 8: beyond the table
    k, v = Dev(be, rng.standard_normal((B, Hkv, D))), Dev(be, rng.standard_normal((B, Hkv, D)))
    ck, cv = Dev(be, np.zeros((12, ps, Hkv, D)), "f16"), Dev(be, np.zeros((12, ps, Hkv, D)), "f16")
    tb, p = i32(be, table), i32(be, pos)
    be.paged_append(s, ck.t, cv.t, k.t, v.t, tb.t, p.t)
    with pytest.raises(ShapeMismatch):
        s.synchronize()
    s.synchronize()                                    # reported once
    want = np.zeros((12, ps, Hkv, D))
    for b in (0, 1, 5):
        want[table[b][pos[b] // ps], pos[b] % ps] = v.f64()[b].astype(np.float16)
    assert np.array_equal(cv.f64(), want)
    ids = i32(be, [0, 6, -1, 1, 2, 3])
    p2 = i32(be, [1, 1, 1, 1, 1, -7])
    be.paged_append(s, ck.t, cv.t, k.t, v.t, tb.t, p2.t, seq_ids=ids.t)
    with pytest.raises(ShapeMismatch):
        ck.t.numpy()
    for t, b in ((0, 0), (3, 1), (4, 2)):
        want[table[b][0], 1] = v.f64()[t].astype(np.float16)
    assert np.array_equal(cv.f64(), want)


# --- attention ----------------------------------------------------------------------------------

def make_cache(be, rng, table_rows, lens, ps, Hkv, D, cache, groups=None, prefix=None, spare=3):
    """Pages in random order; prefixes share their whole pages; what no
    sequence holds is NaN."""
    B = len(lens)
    gs = groups if groups is not None else list(range(B + 1))
    pre = prefix if prefix is not None else [0] * (len(gs) - 1)
    ids = iter(rng.permutation(B * table_rows + spare))
    table = np.zeros((B, table_rows), dtype=np.int32)
    for g in range(len(gs) - 1):
        for b in range(gs[g], gs[g + 1]):
            for i in range(table_rows):
                table[b, i] = table[gs[g], i] if b > gs[g] and (i + 1) * ps <= pre[g] else next(ids)
    for b in range(gs[-1], B):                          # in no group
        for i in range(table_rows):
            table[b, i] = next(ids)
    n = B * table_rows + spare
    ck, cv = np.full((n, ps, Hkv, D), np.nan), np.full((n, ps, Hkv, D), np.nan)
    for b in range(B):
        for p in range(lens[b]):
            at = table[b][p // ps], p % ps
            ck[at], cv[at] = rng.standard_normal((Hkv, D)), rng.standard_normal((Hkv, D))
    return Dev(be, ck, cache), Dev(be, cv, cache), table


def check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache, starts=None, groups=None, prefix=None, scale=None):
    D = q.x.shape[-1]
    scale = float(np.float32(D ** -0.5 if scale is None else scale))
    opt = {n: (None if x is None else i32(be, x)) for n, x in
           (("query_starts", starts), ("group_starts", groups), ("prefix_lens", prefix))}
    tb, ln = i32(be, table), i32(be, lens)
    mark = 12.5
    o = Dev(be, np.full(tuple(q.x.shape), mark), dtype)
    be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, scale, out=o.t, **{n: x and x.t for n, x in opt.items()})
    s.synchronize()
    want, info = ref.attention(q.f64(), ck.f64(), cv.f64(), table, lens, scale, starts, groups, prefix)
    got = o.f64()
    none = np.isnan(want).any((1, 2))
    assert np.array_equal(got[none], np.full_like(got[none], mark))   # rows of no sequence
    close(got[~none], want[~none], ref.attention_bound(want[~none], info[~none], dtype, cache, D))
    return got


PAIRS = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f32")]


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("H,Hkv,D,ps,lens", [
    (32, 4, 64, 16, [257]), (8, 8, 128, 16, [1, 0, 17, 64, 65]), (8, 1, 128, 1, [3, 130]), (14, 2, 64, 24, [100, 1, 63]),
    (4, 1, 80, 7, [40, 129]), (3, 1, 8, 16, [5]), (16, 1, 128, 64, [200, 7]), (40, 2, 128, 32, [90, 33]), (2, 2, 256, 16, [50]),
    (32, 8, 128, 16, [1500, 3, 700])])
def test_attention_single_rows(be, s, dtype, cache, H, Hkv, D, ps, lens):
    rng = np.random.default_rng(H * D + sum(lens))
    rows = -(-max(max(lens), 1) // ps) + 1
    ck, cv, table = make_cache(be, rng, rows, lens, ps, Hkv, D, cache)
    q = Dev(be, rng.standard_normal((len(lens), H, D)) * 2, dtype)
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("H,Hkv,D,ps,lens,groups,prefix", [
    (8, 2, 64, 16, [40, 33, 90, 32], [0, 4], [32]),
    (32, 8, 128, 16, [300, 257, 260, 299, 256], [0, 5], [256]),
    (8, 2, 128, 16, [150, 131, 140, 70, 65, 64, 9], [0, 3, 6, 7], [130, 64, 0]),   # a prefix that ends inside a page
    (4, 4, 64, 8, [20, 10, 5, 30], [0, 3], [16]),      # sequences shorter than the prefix, one in no group
    (16, 1, 64, 32, [700] * 20, [0, 20], [650]),
    (8, 2, 128, 5, [300, 280, 299], [0, 3], [270]),    # pages of no multiple of 8 rows
    (40, 2, 128, 64, [300, 400, 500], [0, 2, 3], [250, 70]),   # many heads, prefixes that end inside a page
    (4, 2, 64, 16, [33, 20, 18], [0, 2, 2, 3], [16, 5, 16]),   # an empty group
])
def test_attention_shared_prefix(be, s, dtype, cache, H, Hkv, D, ps, lens, groups, prefix):
    rng = np.random.default_rng(H + D + sum(lens))
    rows = -(-max(lens) // ps)
    ck, cv, table = make_cache(be, rng, rows, lens, ps, Hkv, D, cache, groups, prefix)
    q = Dev(be, rng.standard_normal((len(lens), H, D)) * 2, dtype)
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache, None, groups, prefix)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("H,Hkv,D,ps,lens,new,groups,prefix", [
    (8, 2, 64, 16, [5], [5], None, None),
    (8, 2, 128, 16, [70, 0, 33, 129], [70, 0, 1, 40], None, None),
    (4, 4, 64, 24, [300], [260], None, None),
    (32, 8, 128, 16, [140, 190, 133], [12, 62, 5], [0, 3], [128]),
    (8, 1, 64, 8, [50, 45, 61, 20], [10, 5, 21, 20], [0, 2, 4], [40, 0]),
    (6, 2, 128, 32, [3, 2], [5, 2], None, None),      # more queries than keys: the first see nothing
    (4, 1, 64, 16, [30, 40], [20, 30], [0, 2], [25]),   # queries inside the prefix
    (8, 1, 64, 16, [200, 260, 170], [60, 100, 33], [0, 3], [130]),   # prompts that fill row blocks, a prefix that ends inside a page
    (8, 2, 128, 32, [400, 333], [300, 200], [0, 2], [128]),
    (8, 2, 128, 8, [300, 290], [150, 140], [0, 2], [140]),
    (8, 2, 80, 24, [300, 290], [150, 140], [0, 2], [144]),
    (8, 2, 128, 10, [300, 290], [150, 140], [0, 2], [77]),    # pages of no multiple of 8 rows
])
def test_attention_many_rows(be, s, dtype, cache, H, Hkv, D, ps, lens, new, groups, prefix):
    rng = np.random.default_rng(H + D + sum(lens) + sum(new))
    rows = -(-max(lens) // ps)
    ck, cv, table = make_cache(be, rng, rows, lens, ps, Hkv, D, cache, groups, prefix)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = Dev(be, rng.standard_normal((starts[-1] + 3, H, D)) * 2, dtype)   # three rows of padding
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache, starts, groups, prefix)


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("B,H,Hkv,D,ps,most,new,shared", [
    (150, 8, 8, 64, 16, 200, 3, False),     # far more row blocks than multiprocessors
    (40, 16, 8, 128, 32, 700, 40, True),    # more than one row tile a block, several blocks a CTA
    (330, 4, 2, 64, 16, 300, 1, True),      # one row each, in groups of eleven
])
def test_attention_many_blocks(be, s, dtype, cache, B, H, Hkv, D, ps, most, new, shared):
    rng = np.random.default_rng(B + H)
    per = 11 if new == 1 else 20
    prefix = 130 if shared else 0
    lens = [int(prefix + max(n, rng.integers(1, most))) for n in [new] * B]
    news = [int(rng.integers(1, new + 1)) for _ in range(B)]
    groups, pre = (list(range(0, B + 1, per)), [prefix] * (B // per)) if shared else (None, None)
    ck, cv, table = make_cache(be, rng, -(-max(lens) // ps), lens, ps, Hkv, D, cache, groups, pre)
    starts = None if new == 1 else np.concatenate([[0], np.cumsum(news)])
    q = Dev(be, rng.standard_normal((B if new == 1 else starts[-1], H, D)) * 2, dtype)
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache, starts, groups, pre)


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_attention_extreme_scores(be, s, dtype, cache):
    """Scores of several thousand (one key takes the whole weight), large
    32-bit queries outside the 16-bit range, and equal scores."""
    rng = np.random.default_rng(12)
    lens, ps, Hkv, D, H = [77, 200, 150], 16, 2, 64, 8
    ck, cv, table = make_cache(be, rng, 13, lens, ps, Hkv, D, cache)
    q = rng.standard_normal((3, H, D))
    q[0] *= 400
    q[1] = 0
    if dtype == "f32":
        q[2, 0] *= 1e6
        q[2, 1] *= 1e-9
    q = Dev(be, q, dtype)
    got = check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache)
    mean = np.array([[cv.f64()[table[1][p // ps], p % ps, h] for p in range(200)] for h in range(Hkv)]).mean(1)
    assert np.abs(got[1].reshape(Hkv, -1, D) - mean[:, None]).max() <= 2.0 ** -7


def test_attention_bad_indices_are_reported(be, s):
    from beacon_cuda import ShapeMismatch
    rng = np.random.default_rng(4)
    lens, ps, Hkv, D, H = [40, 40, 40], 16, 2, 64, 8
    ck, cv, table = make_cache(be, rng, 3, lens, ps, Hkv, D, "f16")
    q = Dev(be, rng.standard_normal((3, H, D)))
    good = check_attention(be, s, rng, q, ck, cv, table, lens, "f32", "f16")

    def run(tab, ln, **more):
        o, tb, l = Dev(be, np.zeros((3, H, D))), i32(be, tab), i32(be, ln)
        keep = {n: i32(be, x) for n, x in more.items()}
        be.paged_attention(s, q.t, ck.t, cv.t, tb.t, l.t, float(np.float32(D ** -0.5)), out=o.t,
                           **{n: x.t for n, x in keep.items()})
        with pytest.raises(ShapeMismatch):
            s.synchronize()
        s.synchronize()
        return o.f64()

    def others_hold(got):
        # the keys may be cut elsewhere; both are within the bound (64 values of
        # at most 4 by 4, scale 1/8; values of at most 5)
        tol = 2 * 5 * (2 * 72 * 2.0 ** -24 * 128 + 2.0 ** -21 + 69 * 2.0 ** -23)
        assert np.abs(got[[0, 2]] - good[[0, 2]]).max() <= tol

    bad = table.copy()
    bad[1, 1] = 1 << 20
    others_hold(run(bad, lens))
    bad[1, 1] = -3
    others_hold(run(bad, lens))
    others_hold(run(table, [40, 1000, 40]))
    others_hold(run(table, [40, -1, 40]))
    run(table, lens, query_starts=[0, 1, 2, 9])
    run(table, lens, group_starts=[0, 7], prefix_lens=[16])
    run(table, lens, group_starts=[0, 3], prefix_lens=[-16])
    assert np.array_equal(check_attention(be, s, rng, q, ck, cv, table, lens, "f32", "f16"), good)


# --- refusals -------------------------------------------------------------------------------------

def refused(status, call):
    from beacon_cuda import EngineError, ShapeMismatch
    from beacon_cuda import _lib as L
    with pytest.raises(EngineError) as e:
        call()
    if status == L.ERR_SHAPE_MISMATCH:
        assert isinstance(e.value, ShapeMismatch)
    else:
        assert e.value.status == status, e.value


def test_rope_refusals(be, s):
    from beacon_cuda import CudaBackend
    from beacon_cuda import _lib as L
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=514), dict(layout=2), dict(scaling=4), dict(scaling=-1),
                dict(theta=1.0), dict(theta=math.nan), dict(factor=2.0), dict(scaling=1, factor=0.5),
                dict(scaling=2, factor=2.0), dict(scaling=3, factor=2.0, original_context=10, low_freq_factor=4.0),
                dict(scaling=2, factor=2.0, original_context=10, beta_slow=0.0), dict(attention_factor=-1.0),
                dict(freq_factors=[0.0] * 32)):
        refused(L.ERR_INVALID_ARGUMENT, lambda: be.rope_create(**{**dict(theta=1e4, rotary_dim=64), **bad}))
    rope = be.rope_create(1e4, 64)
    x, p = be.zeros((2, 3, 64)), be.zeros((2,), L.DTYPE_I32)
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.rope_scaled(s, be.zeros((2, 64)), p, rope))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.rope_scaled(s, be.zeros((2, 3, 32)), p, rope))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.rope_scaled(s, x, be.zeros((3,), L.DTYPE_I32), rope))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.rope_scaled(s, x, be.zeros((2,)), rope))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.rope_scaled(s, be.zeros((2, 3, 64), L.DTYPE_I32), p, rope))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.rope_scaled(s, x, p, rope, out=be.zeros((2, 3, 32))))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.rope_scaled(s, x, p, rope, out=be.zeros((2, 3, 64), L.DTYPE_F16)))
    part = be.wrap(x.device_ptr + 256, (1, 3, 64), L.DTYPE_F32)
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.rope_scaled(s, be.wrap(x.device_ptr, (1, 3, 64), 0),
                                                           be.zeros((1,), L.DTYPE_I32), rope, out=part))
    other = CudaBackend(0)
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.rope_scaled(other.new_stream(), x, p, rope))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.rope_scaled(s, x, p, other.rope_create(1e4, 64)))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.rope_scaled(s, other.zeros((2, 3, 64)), p, rope))
    w = be.zeros((64,))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.qk_norm_rope(s, x, be.zeros((3, 1, 64)), w, w, 1e-5, p, rope))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.qk_norm_rope(s, x, x, be.zeros((32,)), w, 1e-5, p, rope))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.qk_norm_rope(s, x, be.zeros((2, 1, 64), L.DTYPE_F16), w, w, 1e-5, p, rope))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.qk_norm_rope(s, x, x, w, w, -1.0, p, rope))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.qk_norm_rope(s, x, x, w, w, 1e-5, None, rope))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.qk_norm_rope(s, x, x, w, w, 1e-5, p, rope, out_q=x, out_k=x))


def test_append_refusals(be, s):
    from beacon_cuda import _lib as L
    I = L.DTYPE_I32
    ck, cv = be.zeros((4, 8, 2, 64), L.DTYPE_F16), be.zeros((4, 8, 2, 64), L.DTYPE_F16)
    k, tb, p = be.zeros((3, 2, 64)), be.zeros((3, 2), I), be.zeros((3,), I)
    for args in ((ck, be.zeros((4, 8, 2, 64)), k, k, tb, p), (ck, cv, k, be.zeros((2, 2, 64)), tb, p),
                 (ck, cv, be.zeros((3, 1, 64)), be.zeros((3, 1, 64)), tb, p), (ck, cv, k, k, be.zeros((6,), I), p),
                 (ck, cv, k, k, be.zeros((2, 2), I), p), (ck, cv, k, k, tb, be.zeros((2,), I))):
        refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_append(s, *args))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.paged_append(s, be.zeros((4, 8, 2, 64), I), be.zeros((4, 8, 2, 64), I), k, k, tb, p))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.paged_append(s, ck, cv, k, k, be.zeros((3, 2)), p))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_append(s, ck, ck, k, k, tb, p))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_append(s, ck, cv, k, k, tb, p, rope=be.rope_create(1e4, 128)))


def test_attention_refusals(be, s):
    from beacon_cuda import _lib as L
    I, F16 = L.DTYPE_I32, L.DTYPE_F16
    q, ck, cv = be.zeros((3, 4, 64)), be.zeros((4, 8, 2, 64), F16), be.zeros((4, 8, 2, 64), F16)
    tb, ln = be.zeros((3, 2), I), be.zeros((3,), I)
    for args, kw in (((be.zeros((3, 4, 32)), ck, cv, tb, ln), {}), ((be.zeros((3, 3, 64)), ck, cv, tb, ln), {}),
                     ((be.zeros((4, 4, 64)), ck, cv, tb, ln), {}), ((q, ck, be.zeros((4, 8, 1, 64), F16), tb, ln), {}),
                     ((q, ck, cv, be.zeros((6,), I), ln), {}), ((q, ck, cv, tb, be.zeros((2,), I)), {}),
                     ((q, ck, cv, tb, ln), dict(query_starts=be.zeros((3,), I))),
                     ((q, ck, cv, tb, ln), dict(group_starts=be.zeros((2,), I), prefix_lens=be.zeros((2,), I))),
                     ((be.zeros((3, 4, 60)), be.zeros((4, 8, 2, 60), F16), be.zeros((4, 8, 2, 60), F16), tb, ln), {}),
                     ((be.zeros((3, 4, 264)), be.zeros((4, 8, 2, 264), F16), be.zeros((4, 8, 2, 264), F16), tb, ln), {})):
        refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_attention(s, *args, 0.1, **kw))
    for a, b in ((L.DTYPE_F32, L.DTYPE_BF16), (F16, L.DTYPE_F32), (L.DTYPE_BF16, F16), (I, F16)):
        c = be.zeros((4, 8, 2, 64), b)
        refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.paged_attention(s, be.zeros((3, 4, 64), a), c, be.zeros((4, 8, 2, 64), b), tb, ln, 0.1))
    refused(L.ERR_UNSUPPORTED_DTYPE, lambda: be.paged_attention(s, q, ck, cv, tb, be.zeros((3,)), 0.1))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_attention(s, q, ck, cv, tb, ln, math.inf))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_attention(s, q, ck, cv, tb, ln, -0.1))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_attention(s, q, ck, cv, tb, ln, 0.1, out=q))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_attention(s, q, ck, cv, tb, ln, 0.1, prefix_lens=be.zeros((1,), I)))
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_attention(s, q, ck, cv, tb, ln, 0.1, out=be.zeros((3, 4, 32))))
    big = be.zeros((3 * 4 * 64 + 4,))
    refused(L.ERR_INVALID_ARGUMENT, lambda: be.paged_attention(s, be.wrap(big.device_ptr + 4, (3, 4, 64), L.DTYPE_F32), ck, cv, tb, ln, 0.1))


def test_null_arguments(be, s):
    from beacon_cuda import _lib as L
    lib = L.lib()
    for name, n in (("rope_create", 4), ("op_rope_scaled", 6), ("op_qk_norm_rope", 11), ("op_paged_append", 10), ("op_paged_attention", 12)):
        fn = getattr(lib, "beacon_cuda_" + name)
        args = [0.0 if t is ctypes.c_float else None for t in fn.argtypes]
        assert fn(*args) == L.ERR_INVALID_ARGUMENT and len(args) == n
    lib.beacon_cuda_rope_destroy(None)


# --- together --------------------------------------------------------------------------------------

def test_decoding_with_a_shared_prompt(be, s):
    """A prompt is appended once, three continuations share its pages, and six
    steps of norm + rotation, append and attention give what one contiguous
    attention over the same rows gives."""
    rng = np.random.default_rng(21)
    H, Hkv, D, ps, P, B, steps = 8, 2, 64, 16, 37, 3, 6
    rope, freq, _ = make_rope(be, 10000.0, D, "half", "none")
    qw, kw = Dev(be, 1 + 0.1 * rng.standard_normal(D)), Dev(be, 1 + 0.1 * rng.standard_normal(D))
    rows = -(-(P + steps) // ps)
    table = np.zeros((B, rows), dtype=np.int32)
    shared = P // ps
    ids = iter(rng.permutation(shared + B * (rows - shared)))
    table[:, :shared] = [next(ids) for _ in range(shared)]
    for b in range(B):
        table[b, shared:] = [next(ids) for _ in range(rows - shared)]
    n = shared + B * (rows - shared)
    ck, cv = Dev(be, np.full((n, ps, Hkv, D), np.nan), "f16"), Dev(be, np.full((n, ps, Hkv, D), np.nan), "f16")
    tb = i32(be, table)
    scale = float(np.float32(D ** -0.5))
    keys, values = [[] for _ in range(B)], [[] for _ in range(B)]
    f16 = lambda x: x.astype(np.float16).astype(np.float64)
    k0, v0 = rng.standard_normal((P, Hkv, D)), rng.standard_normal((P, Hkv, D))
    # the prompt's rows go to the first sequence; the part of the page that the
    # others own is read through the first as well
    q0 = Dev(be, rng.standard_normal((P, H, D)))
    kd, vd, pos, zero = Dev(be, k0), Dev(be, v0), i32(be, np.arange(P)), i32(be, np.zeros(P))
    qr, kr = be.qk_norm_rope(s, q0.t, kd.t, qw.t, kw.t, 1e-5, pos.t, rope)
    be.paged_append(s, ck.t, cv.t, kr, vd.t, tb.t, pos.t, seq_ids=zero.t)
    starts, ln = i32(be, [0, P, P, P]), i32(be, [P, 0, 0])
    o = be.paged_attention(s, qr, ck.t, cv.t, tb.t, ln.t, scale, query_starts=starts.t).numpy()
    turn = lambda x, w, p: ref.rotate(ref.rms(x, w.f64(), 1e-5), p, freq, True)
    for b in range(B):
        keys[b], values[b] = list(turn(kd.f64(), kw, np.arange(P))), list(f16(vd.f64()))

    def expect(q, b, see):
        K, V = np.array(keys[b])[:see], np.array(values[b])[:see]
        out = np.zeros((H, D))
        for h in range(H):
            x = K[:, h // (H // Hkv)] @ q[h] * scale
            p = np.exp(x - x.max())
            out[h] = p / p.sum() @ V[:, h // (H // Hkv)]
        return out

    qq = turn(q0.f64(), qw, np.arange(P))
    # the keys are kept in 16 bits: a score moves by 2^-11 of its sum of
    # magnitudes (below 64 here: 64 values of at most 4 by 2, scale 1/8)
    tol = 2 * 64 * 2.0 ** -11
    for t in (0, 1, 16, P - 1):
        assert np.abs(o[t] - expect(qq[t], 0, t + 1)).max() <= tol
    gs, pl = i32(be, [0, B]), i32(be, [P])
    for step in range(steps):
        p = np.full(B, P + step)
        q, k, v = Dev(be, rng.standard_normal((B, H, D))), Dev(be, rng.standard_normal((B, Hkv, D))), Dev(be, rng.standard_normal((B, Hkv, D)))
        pd, ld = i32(be, p), i32(be, p + 1)
        be.qk_norm_rope(s, q.t, k.t, qw.t, kw.t, 1e-5, out_q=q.t, out_k=k.t)
        qd = Dev(be, np.zeros((B, H, D)))
        be.rope_scaled(s, q.t, pd.t, rope, out=qd.t)
        be.paged_append(s, ck.t, cv.t, k.t, v.t, tb.t, pd.t, rope=rope)
        o = be.paged_attention(s, qd.t, ck.t, cv.t, tb.t, ld.t, scale, group_starts=gs.t, prefix_lens=pl.t).numpy()
        for b in range(B):
            # k was normalised in place: its values are the device's own
            keys[b].append(ref.rotate(k.f64()[b:b + 1], p[b:b + 1], freq, True)[0])
            values[b].append(f16(v.f64()[b]))
            assert np.abs(o[b] - expect(qd.f64()[b], b, P + step + 1)).max() <= tol, (step, b)


def test_captured_calls_replay(be, torch_):
    """Two graphs captured on one stream replay, alternately and overlapping on
    two streams, with the lengths and rows of the moment; a graph holds its own
    scratch."""
    torch = torch_
    rng = np.random.default_rng(31)
    H, Hkv, D, ps, B = 32, 8, 128, 16, 4
    lens = [900, 640, 513, 777]
    cases = []
    side = torch.cuda.Stream()
    s = be.wrap_stream(side.cuda_stream)
    for prefix in (None, [512]):
        groups = None if prefix is None else [0, B]
        ck, cv, table = make_cache(be, rng, 57, lens, ps, Hkv, D, "f16", groups, prefix)
        q, o = Dev(be, rng.standard_normal((B, H, D))), Dev(be, np.zeros((B, H, D)))
        tb, ln = i32(be, table), i32(be, lens)
        gs, pl = (None, None) if prefix is None else (i32(be, groups), i32(be, prefix))
        kw = dict(group_starts=gs and gs.t, prefix_lens=pl and pl.t, out=o.t)
        args = (q.t, ck.t, cv.t, tb.t, ln.t, float(np.float32(D ** -0.5)))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            be.paged_attention(s, *args, **kw)
        cases.append((g, q, o, ln, ck, cv, table, groups, prefix, (tb, gs, pl)))
    for rnd in range(4):
        cut = [max(513, x - 40 * rnd) for x in lens]
        qs = [rng.standard_normal((B, H, D)) for _ in cases]
        for (g, q, o, ln, *_), x in zip(cases, qs):
            q.x.copy_(torch.as_tensor(x))
            ln.x.copy_(torch.as_tensor(np.array(cut, dtype=np.int32)))
            o.x.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for k, (g, *_) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                g.replay()
        torch.cuda.synchronize()
        for g, q, o, ln, ck, cv, table, groups, prefix, _ in cases:
            want, info = ref.attention(q.f64(), ck.f64(), cv.f64(), table, cut, float(np.float32(D ** -0.5)), None, groups, prefix)
            close(o.f64(), want, ref.attention_bound(want, info, "f32", "f16", D), f"round {rnd}")


def test_two_streams_at_once(be, torch_):
    """Calls on two streams share nothing but their inputs."""
    rng = np.random.default_rng(32)
    H, Hkv, D, ps = 32, 8, 128, 16
    lens = [2000, 1500]
    ck, cv, table = make_cache(be, rng, 125, lens, ps, Hkv, D, "f16")
    tb, ln = i32(be, table), i32(be, lens)
    streams = [be.new_stream(), be.new_stream()]
    qs = [Dev(be, rng.standard_normal((2, H, D))) for _ in range(2)]
    outs = [[], []]
    for _ in range(8):
        for k in range(2):
            outs[k].append(be.paged_attention(streams[k], qs[k].t, ck.t, cv.t, tb.t, ln.t, 0.1))
    for k in range(2):
        want, info = ref.attention(qs[k].f64(), ck.f64(), cv.f64(), table, lens, float(np.float32(0.1)))
        for o in outs[k]:
            close(o.numpy().astype(np.float64), want, ref.attention_bound(want, info, "f32", "f16", D))


@pytest.mark.parametrize("new,ps", [(1, 16), (40, 16), (40, 7)])
def test_attention_wait_timeout_is_reported(be, new, ps):
    """A bounded wait that runs out is reported as such, and the stream works on."""
    from beacon_cuda import EngineError
    from beacon_cuda import _lib as L
    rng = np.random.default_rng(33)
    H, Hkv, D, lens = 32, 8, 128, [6000, 4100, 5000, 300]
    B = len(lens)
    ck, cv, table = make_cache(be, rng, -(-max(lens) // ps), lens, ps, Hkv, D, "f16")
    starts = None if new == 1 else [new * i for i in range(B + 1)]
    q = Dev(be, rng.standard_normal((B * new, H, D)), "f16")
    tb, ln, st = i32(be, table), i32(be, lens), starts and i32(be, starts)
    s = be.new_stream()
    statuses = []
    be.set_wait_limit(1)
    try:
        for _ in range(20):
            be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 0.1, query_starts=st and st.t)
            try:
                s.synchronize()
                statuses.append(L.OK)
            except EngineError as e:
                statuses.append(e.status)
                break
    finally:
        be.set_wait_limit(0)
    assert L.ERR_DEVICE_TIMEOUT in statuses, statuses
    for _ in range(2):
        check_attention(be, s, rng, q, ck, cv, table, lens, "f16", "f16", starts)


def test_attention_without_pages(be, s):
    """A cache without pages, or a table without entries, holds no key: zeros; a length then is an error."""
    from beacon_cuda import ShapeMismatch
    from beacon_cuda import _lib as L
    rng = np.random.default_rng(34)
    some = Dev(be, np.zeros(16), "f16")
    for pages, max_pages in ((0, 2), (3, 0), (0, 0)):
        full = Dev(be, np.zeros((3, 16, 2, 64)), "f16")
        cache = full.t if pages else be.wrap(some.x.data_ptr(), (0, 16, 2, 64), L.DTYPE_F16)
        entries = i32(be, np.zeros((3, 2)))
        table = entries.t if max_pages else be.wrap(some.x.data_ptr(), (3, 0), L.DTYPE_I32)
        q, o = Dev(be, rng.standard_normal((3, 8, 64))), Dev(be, np.ones((3, 8, 64)))
        lens = i32(be, [0, 0, 0])
        be.paged_attention(s, q.t, cache, cache, table, lens.t, 1.0, out=o.t)
        s.synchronize()
        assert not o.f64().any()
        lens = i32(be, [1, 0, 0])
        be.paged_attention(s, q.t, cache, cache, table, lens.t, 1.0, out=o.t)
        with pytest.raises(ShapeMismatch):
            s.synchronize()


def test_attention_on_the_default_stream(be):
    rng = np.random.default_rng(35)
    lens = [300, 40, 300]
    s = be.wrap_stream(0)
    ck, cv, table = make_cache(be, rng, 20, lens, 16, 2, 128, "bf16", [0, 3], [32])
    q = Dev(be, rng.standard_normal((3, 8, 128)), "bf16")
    check_attention(be, s, rng, q, ck, cv, table, lens, "bf16", "bf16", None, [0, 3], [32])


def test_two_threads_on_one_stream(be):
    """Calls of several launches from two threads do not mix."""
    import threading
    rng = np.random.default_rng(36)
    H, Hkv, D, ps = 32, 8, 128, 16
    s = be.new_stream()
    jobs = []
    for lens in ([900, 800, 700, 650], [40, 500, 300, 513]):
        m = min(lens) // 2
        ck, cv, table = make_cache(be, rng, 57, lens, ps, Hkv, D, "f16", [0, 4], [m])
        q = Dev(be, rng.standard_normal((4, H, D)), "f16")
        outs = [Dev(be, np.zeros((4, H, D)), "f16") for _ in range(50)]
        jobs.append((q, ck, cv, table, lens, m, i32(be, table), i32(be, lens), i32(be, [0, 4]), i32(be, [m]), outs))

    def work(j):
        q, ck, cv, _, _, _, tb, ln, gs, pl, outs = j
        for o in outs:
            be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 0.1, group_starts=gs.t, prefix_lens=pl.t, out=o.t)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    s.synchronize()
    for q, ck, cv, table, lens, m, *_, outs in jobs:
        want, info = ref.attention(q.f64(), ck.f64(), cv.f64(), table, lens, float(np.float32(0.1)), None, [0, 4], [m])
        bound = ref.attention_bound(want, info, "f16", "f16", D)
        for o in outs:
            close(o.f64(), want, bound)
