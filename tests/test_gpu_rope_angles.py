"""Sines and cosines of the rotation, at angles where one of them is small."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import Dev, be, i32, s  # noqa: F401 (be, s: fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_small_sines_and_cosines(be, s, layout):
    """A pair (1, 0) turns to (cos, sin): each within 2 steps of 32 bits of the
    true value (one of sincospi, a half of the remainder's sum, a half spare).
    The angle itself is known to 2e5 2^-51 (the product of the position and a
    64-bit frequency, off by two steps)."""
    from beacon_cuda import _lib as L
    D, T = 128, 4096
    rope = be.rope_create(10000.0, D, L.ROPE_HALF if layout == "half" else L.ROPE_INTERLEAVED)
    pos = np.random.default_rng(51).integers(0, 200000, T)
    x = np.zeros((T, 1, D))
    first, second = (np.s_[..., :D // 2], np.s_[..., D // 2:]) if layout == "half" else (np.s_[..., 0::2], np.s_[..., 1::2])
    x[first] = 1.0
    xd, p, o = Dev(be, x), i32(be, pos), Dev(be, np.zeros((T, 1, D)))
    be.rope_scaled(s, xd.t, p.t, rope, out=o.t)
    s.synchronize()
    angle = pos[:, None, None] * ref.frequencies(10000.0, D)
    for part, want in ((first, np.cos(angle)), (second, np.sin(angle))):
        off = np.abs(o.f64()[part] - want)
        bound = 2 * np.spacing(np.abs(want).astype(np.float32)).astype(np.float64) + 2e5 * 2.0 ** -51
        assert (off <= bound).all(), (off / bound).max()
