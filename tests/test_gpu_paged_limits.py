"""The largest page tables and row numbers of paged attention."""
import numpy as np
import pytest

from test_gpu_paged import Dev, be, check_attention, i32, refused, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
def test_wide_page_tables(be, s, dtype, cache):
    """Tables with room for up to 2^31 - 4096 positions work; kernels would count
    past 32 bits in wider ones, which are refused."""
    from beacon_cuda import _lib as L
    rng = np.random.default_rng(71)
    ps, D, lens = 1 << 16, 8, [300, 70]
    ck, cv = (Dev(be, rng.standard_normal((2, ps, 1, D)), cache) for _ in range(2))
    q = Dev(be, rng.standard_normal((2, 4, D)), dtype)
    table = np.zeros((2, (1 << 15) - 1), dtype=np.int32)
    table[1, 0] = 1
    check_attention(be, s, rng, q, ck, cv, table, lens, dtype, cache)
    wide, ln = i32(be, np.zeros((2, 1 << 15))), i32(be, lens)
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_attention(s, q.t, ck.t, cv.t, wide.t, ln.t, 1.0))


def test_row_numbers(be, s):
    """(Refused before anything is read: the tensors' memory is not there.)"""
    from beacon_cuda import _lib as L
    n = 0x3FFFFFFF
    x, c = Dev(be, np.zeros(64), "f16"), Dev(be, np.zeros((1, 16, 1, 8)), "f16")
    wrap = lambda shape, kind: be.wrap(x.x.data_ptr(), shape, kind)
    q, out = wrap((n, 2, 8), L.DTYPE_F16), wrap((n, 2, 8), L.DTYPE_F16)
    refused(L.ERR_SHAPE_MISMATCH, lambda: be.paged_attention(s, q, c.t, c.t, wrap((n, 1), L.DTYPE_I32), wrap((n - 1,), L.DTYPE_I32), 1.0,
                                                             out=out))
