"""Step sizes held to limits of either sign."""
import numpy as np
import pytest

from layer_ref import BF16, F16, F32, Layer, check_scan, elt_dtype, from_type, scan
from nextsycl_amd import DevBuf
from test_gpu_ssm_edges import E, Call, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("rate,lo,hi", [(-1.0, -np.inf, -0.03), (0.5, -0.1, -0.1), (-1.0, -2.0, 0.0), (-1.0, -1.0, 0.01)])
def test_limits_of_either_sign(ops, qt, T, rate, lo, hi):
    """A step is softplus held to lo .. hi, which may be below 0 and leave it negative: a decay that grows, an outer product subtracted."""
    H, P, N, G, K = 4, 20, 64, 2, 4
    L = Layer(H, P, N, G, K, seed=41, rate=rate)
    raw, val = rows_of(L, qt, T, 42)
    L.d = None
    y, h, yb, hb = scan(L, val[:, :L.chan], val[:, L.chan:], np.zeros((K - 1, L.chan)), np.zeros((H, P, N)), lo, hi)
    # (steps are of one sign: of negative ones the bounds are sums of negative sizes)
    yb, hb = np.abs(yb), np.abs(hb)
    c = Call(ops, L, qt, raw)
    e, row = E[qt], L.chan + H
    ops.ssm_prompt(qt, c.rows, row, c.rows.view(L.chan * e, c.rows.len - L.chan * e), row, *c.w, c.ring, 4, 0, T, H, P, N, G, K, None, c.h, c.y, L.inner, c.sc, dt_lo=lo, dt_hi=hi)
    got, state = c.out()
    check_scan(got, y, yb, qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")


def test_a_slot_whose_first_position_is_negative_is_passed_over(ops):
    g, H, P, N, K, cap = ops.gpu, 2, 8, 16, 4, 7
    L = Layer(H, P, N, 1, K, seed=43)
    raw, val = rows_of(L, F32, 3, 44)
    ring = np.random.default_rng(45).standard_normal((2, cap, L.chan)).astype(np.float32)
    h0 = np.random.default_rng(46).standard_normal((2, H, P, N)).astype(np.float32)
    w = [DevBuf.of(g, a) for a in (L.cw, L.cb, L.a, L.dtb, L.d)]
    rows, ringb, h0b, h1b, y, row = DevBuf.of(g, raw), DevBuf.of(g, ring), DevBuf.of(g, h0), DevBuf(g, h0.nbytes), DevBuf(g, 3 * L.inner * 4), L.chan + H
    h1b.fill(0xFF)
    y.fill(0xFF)
    ops.ssm_step(F32, rows, row, rows.view(L.chan * 4, rows.len - L.chan * 4), row, *w, ringb, cap, 0, 3, H, P, N, 1, K, h0b, h1b, y, L.inner, nslots=2,
                 slots=DevBuf.of(g, np.array([1, 0, 1], np.int32)), pos=DevBuf.of(g, np.array([-1, 5, 0], np.int32)))
    got = y.read(np.uint32).reshape(3, -1)
    assert (got[[0, 2]] == 0xFFFFFFFF).all() and (h1b.read(np.uint32).reshape(2, -1)[1] == 0xFFFFFFFF).all() and np.array_equal(ringb.read(np.float32).reshape(ring.shape)[1], ring[1])
    r, h, rb, hb = scan(L, val[1:2, :L.chan], val[1:2, L.chan:], ring[0][np.arange(2, 5) % cap], h0[0])
    check_scan(got[1:2].view(np.float32), r, rb, F32, 1, N, "the other slot")
