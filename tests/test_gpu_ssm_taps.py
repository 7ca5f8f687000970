"""Convolutions of fewer than 4 taps: a value that is not finite reaches the rows whose taps hold it and none behind them."""
import numpy as np
import pytest

from layer_ref import BF16, F16, F32, Layer, check_scan, elt_dtype, from_type, to_type
from nextsycl_amd import DevBuf
from test_gpu_ssm_edges import E, Call, plain, rows_of

pytestmark = pytest.mark.gpu


# T, the ring's rows, rows a call (steps: of that many rows; 0: a prompt)
@pytest.mark.parametrize("T,cap,each", [(150, 4, 0), (12, 40, 0), (12, 8, 4), (12, 8, 1)])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
@pytest.mark.parametrize("qt,bad", [(F32, np.inf), (F16, np.nan), (BF16, -np.inf)])
def test_c_that_is_not_finite_in_one_row(ops, qt, bad, K, T, cap, each):
    H, P, N, G = 4, 20, 64, 2
    L = Layer(H, P, N, G, K, seed=31)
    raw, val = rows_of(L, qt, T, 32)
    y, h, yb, hb = plain(L, val)
    at = 62 if T > 64 else 5                       # (its taps end in the next chunk, or in the next call)
    spoilt = val.copy()
    spoilt[at, L.inner + (G + 1) * N + 9] = bad    # of the second group's C
    g, e, row = ops.gpu, E[qt], L.chan + H
    c = Call(ops, L, qt, to_type(qt, spoilt)[0])
    ring = DevBuf.of(g, np.full((cap, L.chan), np.nan, np.float32))
    if each:
        c.h.fill(0)
        for t in range(0, T, each):
            at_ = lambda o: c.rows.view((t * row + o) * e, c.rows.len - (t * row + o) * e)  # noqa: E731,B023
            ops.ssm_step(qt, at_(0), row, at_(L.chan), row, *c.w, ring, cap, t, each, H, P, N, G, K, c.h, c.h, c.y.view(t * L.inner * e, each * L.inner * e), L.inner,
                         slots=DevBuf.of(g, np.zeros(each, np.int32)))
            g.sync()
    else:
        ops.ssm_prompt(qt, c.rows, row, c.rows.view(L.chan * e, c.rows.len - L.chan * e), row, *c.w, ring, cap, 0, T, H, P, N, G, K, None, c.h, c.y, L.inner, c.sc)
    got, state = c.out()
    lost = np.zeros((T, H, P), bool)
    lost[at:at + K, 2:] = True
    lost = lost.reshape(T, -1)
    assert not np.isfinite(got[lost]).any()
    check_scan(got[~lost][None], y[~lost][None], yb[~lost][None], qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")
