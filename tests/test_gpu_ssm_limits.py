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
