"""The norms and 4-bit products at the most that one call takes: every row is there."""
import numpy as np
import pytest

from layer_ref import F32, q4_weights
from nextsycl_amd import DevBuf, Error

pytestmark = pytest.mark.gpu


def test_norm_of_the_most_rows(ops):
    g, T = ops.gpu, (1 << 26) - 4
    r = np.random.default_rng(1)
    x, h = r.standard_normal(T, np.float32), r.standard_normal(T, np.float32)
    xb, hb, out = DevBuf.of(g, x), DevBuf.of(g, h), DevBuf(g, 4 * T)
    ops.norm_residual(F32, F32, xb, 1, hb, 1, out, 1, None, 0, T, 1, 1e-5)
    assert np.array_equal(out.read(np.float32), h + x)
    with pytest.raises(Error, match="too many rows"):
        big = DevBuf(g, 4 * (T + 1))
        ops.norm_residual(F32, F32, big, 1, big, 1, big, 1, None, 0, T + 1, 1, 1e-5)


def test_4_bit_product_of_the_most_outputs(ops):
    """Weights of 0 but for the last tile."""
    g, M, K, group = ops.gpu, (1 << 27) - 16, 5, 128
    w = DevBuf(g, ops.q4_bytes(M, K, group))
    w.fill(0x88)
    r = np.random.default_rng(2)
    last = np.concatenate([r.integers(0, 256, 1024, np.uint8), r.uniform(0.01, 0.1, 16).astype(np.float16).view(np.uint8)])
    w.view(w.len - last.nbytes, last.nbytes).write(last)
    x = r.standard_normal(K).astype(np.float32)
    y = DevBuf(g, 4 * M)
    ops.q4_product(F32, DevBuf.of(g, x), K, w, group, y, M, 1, M, K)
    got = y.read(np.float32)
    want = q4_weights(last, 16, 128, group)[0][:, :K]
    # (5 products of 22 bits, summed in float32)
    assert (np.abs(got[-16:] - want @ x) <= 2.0 ** -21 * (np.abs(want) @ np.abs(x))).all() and not got[:-16].any()
