"""Paged attention on streams that other operators use at the same time, and
the scratch that a stream keeps for it."""
import threading

import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import Dev, be, check_attention, close, i32, make_cache, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [None, 3])
@pytest.mark.parametrize("rows", [1, 16, 200])
def test_beside_matrix_products_of_another_thread(be, rows, new):
    """One thread attends, one multiplies by quantised weights, on one stream:
    neither's partial results are in the other's way."""
    import oracle as orc
    from beacon_cuda import _lib as L
    rng = np.random.default_rng(61)
    H, Hkv, D, ps, lens = 32, 8, 128, 16, [900, 800, 700, 650]
    ck, cv, table = make_cache(be, rng, 57, lens, ps, Hkv, D, "f16", [0, 4], [600])
    starts = None if new is None else np.arange(5) * new
    q = Dev(be, rng.standard_normal((4 * (new or 1), H, D)), "f16")
    tb, ln, gs, pl = i32(be, table), i32(be, lens), i32(be, [0, 4]), i32(be, [600])
    st = None if starts is None else i32(be, starts)
    outs = [Dev(be, np.zeros(tuple(q.x.shape)), "f16") for _ in range(100)]
    n, k = 512, 8192
    w = be.upload(orc.quantize((rng.standard_normal((n, k)) * 0.02).astype(np.float32), orc.Q4_K), shape=(n, k), dtype=L.DTYPE_Q4_K)
    x = be.upload(rng.standard_normal((rows, k)).astype(np.float32))
    s = be.new_stream()
    alone = be.quantized_matmul(s, x, w).numpy()     # also makes its scratch
    assert np.array_equal(alone, be.quantized_matmul(s, x, w).numpy())
    products = []

    def attend():
        for o in outs:
            be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 0.1, query_starts=st and st.t, group_starts=gs.t, prefix_lens=pl.t,
                               out=o.t)

    def multiply():
        for _ in range(100):
            products.append(be.quantized_matmul(s, x, w))

    threads = [threading.Thread(target=f) for f in (attend, multiply)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    s.synchronize()
    for p in products:
        assert np.array_equal(p.numpy(), alone)
    want, info = ref.attention(q.f64(), ck.f64(), cv.f64(), table, lens, float(np.float32(0.1)), starts, [0, 4], [600])
    bound = ref.attention_bound(want, info, "f16", "f16", D)
    for o in outs:
        close(o.f64(), want, bound)


@pytest.mark.parametrize("wrapped", [False, True])
def test_growing_calls_and_the_end_of_a_stream(be, wrapped):
    """Calls that need more scratch each time, back to back, and a stream that
    is let go right behind its last call."""
    import torch
    rng = np.random.default_rng(62)
    H, Hkv, D, ps = 32, 8, 128, 16
    jobs = []
    for B in (1, 3, 20, 40):
        lens = [300 + 7 * b for b in range(B)]
        ck, cv, table = make_cache(be, rng, 40, lens, ps, Hkv, D, "f16", [0, B], [200])
        q = Dev(be, rng.standard_normal((B, H, D)), "f16")
        jobs.append((q, ck, cv, table, lens, i32(be, table), i32(be, lens), i32(be, [0, B]), i32(be, [200]),
                     Dev(be, np.zeros((B, H, D)), "f16")))
    side = torch.cuda.Stream()
    s = be.wrap_stream(side.cuda_stream) if wrapped else be.new_stream()
    for q, ck, cv, _, _, tb, ln, gs, pl, o in jobs + jobs[::-1]:
        be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 0.1, group_starts=gs.t, prefix_lens=pl.t, out=o.t)
    del s
    torch.cuda.synchronize()
    for q, ck, cv, table, lens, *_, o in jobs:
        want, info = ref.attention(q.f64(), ck.f64(), cv.f64(), table, lens, float(np.float32(0.1)), None, [0, len(lens)], [200])
        close(o.f64(), want, ref.attention_bound(want, info, "f16", "f16", D))


def test_scratch_goes_back(be):
    """A stream's scratch for a large call is the device's again when the stream ends."""
    import torch
    rng = np.random.default_rng(63)
    B, H, Hkv, D, ps = 512, 64, 8, 128, 16
    table = np.zeros((B, 4))
    ck = Dev(be, rng.standard_normal((4, ps, Hkv, D)), "f16")
    q, tb, ln = Dev(be, np.zeros((B, H, D)), "f16"), i32(be, table), i32(be, np.full(B, 40))
    gs, pl, o = i32(be, [0, B]), i32(be, [32]), Dev(be, np.zeros((B, H, D)), "f16")
    free = []
    for _ in range(6):
        s = be.new_stream()
        be.paged_attention(s, q.t, ck.t, ck.t, tb.t, ln.t, 0.1, group_starts=gs.t, prefix_lens=pl.t, out=o.t)
        s.synchronize()
        del s
        torch.cuda.synchronize()
        free.append(torch.cuda.mem_get_info()[0])
    assert free[-1] >= free[0] - (8 << 20)            # 32 MB of sums a call


def test_first_calls_of_many_threads(be):
    """Threads that use a new stream at once share its error words: an index out
    of range in one of their calls is reported, once."""
    from beacon_cuda import ShapeMismatch
    rng = np.random.default_rng(64)
    k = Dev(be, rng.standard_normal((1, 2, 64)))
    tb, good, bad = i32(be, [[0, 1]]), i32(be, [3]), i32(be, [99])
    caches = [(Dev(be, np.zeros((2, 4, 2, 64)), "f16"), Dev(be, np.zeros((2, 4, 2, 64)), "f16")) for _ in range(8)]
    for rnd in range(20):
        s = be.new_stream()
        gate = threading.Barrier(8)

        def work(i):
            gate.wait()
            be.paged_append(s, caches[i][0].t, caches[i][1].t, k.t, k.t, tb.t, (bad if i == rnd % 8 else good).t)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        with pytest.raises(ShapeMismatch):
            s.synchronize()
        s.synchronize()


@pytest.mark.parametrize("new", [None, 2])
def test_inputs_that_change_on_the_stream(be, new):
    """Queries, lengths, tables and cache rows written by kernels right before
    each call, with no wait between: every call reads what stands there then."""
    import torch
    rng = np.random.default_rng(65)
    H, Hkv, D, ps, B, N = 32, 8, 128, 16, 6, 60
    lens = [700, 640, 513, 777, 600, 530]
    ck, cv, table = make_cache(be, rng, 50, lens, ps, Hkv, D, "f16", [0, B], [512])
    for c in (ck, cv):
        c.x.nan_to_num_()
    side = torch.cuda.Stream()
    s = be.wrap_stream(side.cuda_stream)
    T = B * (new or 1)
    q, tb, ln = Dev(be, np.zeros((T, H, D)), "f16"), i32(be, table), i32(be, lens)
    gs, pl = i32(be, [0, B]), i32(be, [512])
    st = None if new is None else i32(be, np.arange(B + 1) * new)
    qs = torch.randn(N, T, H, D, device="cuda").half()
    ls = torch.tensor(np.array([[max(513, x - int(rng.integers(0, 200))) for x in lens] for _ in range(N)], dtype=np.int32), device="cuda")
    rows = torch.randn(N, Hkv, D, device="cuda").half()
    first = [int(table[0, 3]), 5]                      # a key of the prefix

    def step(i, out):
        q.x.copy_(qs[i])
        ln.x.copy_(ls[i])
        ck.x[first[0], first[1]] = rows[i]
        cv.x[first[0], first[1]] = rows[i]
        be.paged_attention(s, q.t, ck.t, cv.t, tb.t, ln.t, 0.1, query_starts=st and st.t, group_starts=gs.t, prefix_lens=pl.t, out=out.t)

    outs = [[Dev(be, np.zeros((T, H, D)), "f16") for _ in range(N)] for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in range(N):
            step(i, outs[0][i])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in range(N):
            torch.cuda.synchronize()
            step(i, outs[1][i])
    s.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a.x, b.x)
    for i in (0, N - 1):
        q.x.copy_(qs[i])
        for c in (ck, cv):
            c.x[first[0], first[1]] = rows[i]
        starts = None if new is None else np.arange(B + 1) * new
        args = (q.f64(), ck.f64(), cv.f64(), table, ls[i].cpu().numpy(), float(np.float32(0.1)), starts, [0, B], [512])
        want, info = ref.attention(*args)
        close(outs[0][i].f64(), want, ref.attention_bound(want, info, "f16", "f16", D))
