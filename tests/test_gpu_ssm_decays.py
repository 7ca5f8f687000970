"""ns_ssm_prompt where steps of very different sizes stand side by side: what a row leaves behind decays by the steps between, however large the
row's own is. Against the definition row by row in float64, and against ns_ssm_step."""
import numpy as np
import pytest

from layer_ref import BF16, F16, F32, ROUND, TINY, Layer, check_scan, elt_dtype, from_type, scan_tolerance, to_type
from nextsycl_amd import DevBuf
from test_gpu_ssm_edges import E, Call, plain

pytestmark = pytest.mark.gpu


def near(got, ref, bound, qt, T, N, what):
    """check_scan for operands of 22 bits whatever the rows' type: float32 arithmetic and the output's own rounding, nothing beside them
    (bfloat16 rows: check_scan's, their operands may be halfs)."""
    check_scan(got, ref, bound, qt, T, N, what)
    if qt == BF16:
        return
    err, tol = np.abs(got.astype(np.float64) - ref), scan_tolerance(T, N) * bound + ROUND[qt] * np.abs(ref) + TINY[qt]
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), "%s: %s is %.9g, should be %.9g, off by %.3g of %.3g" % (what, at, got[at], ref[at], err[at], tol[at])
    # (root mean square: roundings of either sign, and the output's of half a step at most)
    rel = np.linalg.norm(err) / np.linalg.norm(ref)
    assert rel <= 2.0 ** -18 + (ROUND[qt] if qt != F32 else 0.0), "%s: relative error %.3g" % (what, rel)


def rows_with_steps(L, qt, steps, seed):
    """x, B and C positive (nothing cancels: an error of a decay is one of y); a row's step much the same for every head, softplus the identity of
    the large ones."""
    T = len(steps)
    v = np.random.default_rng(seed).standard_normal((T, L.chan + L.H))
    v[:, :L.chan] = 0.05 + 0.08 * np.abs(v[:, :L.chan])
    L.cw = np.abs(L.cw)
    if L.cb is not None:
        L.cb = np.abs(L.cb)
    s = np.asarray(steps)[:, None]
    v[:, L.chan:] = s + np.where(s > 1.0, 0.0, 0.5) * v[:, L.chan:]
    return to_type(qt, v)


def large_among_small(size, T=150):
    steps = np.full(T, -4.0)
    steps[[5, 37, 38, 71, 127]] = size                # in the middle of runs of 16, in runs in front of others, side by side, at a chunk's end
    return steps


STEPS = {"50": large_among_small(50.0), "1000": large_among_small(1000.0), "60000": large_among_small(60000.0),
         "20 in front of 0.01": np.where(np.arange(150) % 16 < 8, 20.0, -4.6), "spread": 3.0 * np.random.default_rng(1).standard_normal(150) - 2.0}


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("name", list(STEPS))
def test_rows_behind_a_large_step(ops, qt, name):
    H, P, N, G, K = 4, 40, 64, 2, 4
    L = Layer(H, P, N, G, K, seed=21, rate=-16.0)
    L.dtb = None
    raw, val = rows_with_steps(L, qt, STEPS[name], 22)
    T = raw.shape[0]
    y, h, yb, hb = plain(L, val)
    c = Call(ops, L, qt, raw)
    c.run()
    got, state = c.out()
    near(got, y, yb, qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")
    # each row by its own size: the large step's rows would hide what the others lose
    rel = np.linalg.norm(got - y, axis=1) / np.linalg.norm(y, axis=1)
    assert (rel <= 2.0 ** -18 + (3 * 2.0 ** -11 if qt == BF16 else 0.0) + (ROUND[qt] if qt != F32 else 0.0)).all(), rel.max()
    # row by row
    g, e, row = ops.gpu, E[qt], L.chan + L.H
    ring, st, one = DevBuf.of(g, np.full((4, L.chan), np.nan, np.float32)), DevBuf.of(g, np.zeros((H, P, N), np.float32)), DevBuf(g, T * L.inner * e)
    at = lambda t, o: c.rows.view((t * row + o) * e, c.rows.len - (t * row + o) * e)  # noqa: E731
    for t in range(T):
        ops.ssm_step(qt, at(t, 0), row, at(t, L.chan), row, *c.w, ring, 4, t, 1, H, P, N, G, K, st, st, one.view(t * L.inner * e, L.inner * e), L.inner)
    steps = from_type(qt, one.read(elt_dtype(qt)).reshape(T, -1))
    near(steps, y, yb, qt, T, N, "steps")


def test_a_decay_keeps_its_bits_behind_a_large_step(ops):
    """One feature, B and C and x of 1, a row with a step of 1000 and then rows with steps of 1 / 64: y of a row behind it is, but for 2^-13 of it, the
    large row's 1000 times the decay, whose exponent is 16 / 64 a row. Within 2^-18 (in 2^-24: the exponent, 4.25 at most, within 4 roundings of
    itself, 17; three silu and an exponential, 12; two operands of 22 bits, 8; the sums, 4)."""
    H, P, N, T = 1, 1, 1, 32
    L = Layer(H, P, N, 1, 1, seed=0, bias=False, rate=-16.0)
    L.cw[:] = 1.0
    raw = np.zeros((T, L.chan + H), np.float32)
    raw[:, :L.chan] = 1.2784645                          # silu of it is 1 within 2^-22
    raw[:, L.chan:] = np.log(np.expm1(1.0 / 64))
    raw[3, L.chan] = 1000.0
    y, h, yb, hb = plain(L, raw)
    c = Call(ops, L, F32, raw)
    c.run()
    got, state = c.out()
    assert (np.abs(got - y)[3:20] <= 2.0 ** -18 * np.abs(y)[3:20]).all(), (np.abs(got - y) / np.abs(y))[3:20].max()


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("size", [1e9, 1e30])
def test_steps_past_any_decay(ops, qt, size):
    """A step so large that sums of 64 bits lose the others beside it: nothing of the rows in front of it is left, and what it leaves itself decays by the
    steps behind it."""
    H, P, N, G, K, T, at = 2, 16, 32, 1, 1, 100, 41
    L = Layer(H, P, N, G, K, seed=23, bias=False, rate=-4.0)
    raw, val = rows_with_steps(L, qt, np.where(np.arange(T) == at, size, -3.0), 24)
    y, h, yb, hb = plain(L, val)
    c = Call(ops, L, qt, raw)
    c.run()
    got, state = c.out()
    for part in (slice(0, at), slice(at, 50), slice(50, 64), slice(64, T)):       # (y falls by 10 powers of ten behind it)
        near(got[part], y[part], yb[part], qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")
