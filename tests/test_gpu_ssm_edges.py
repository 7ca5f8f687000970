"""ns_ssm_prompt where it can go wrong: values that are not finite, wide ranges of values in a column, long prompts of wide
states in segments and passes, prompts recorded into graphs, two prompts at once on two handles."""
import ctypes as C

import numpy as np
import pytest

from layer_ref import BF16, F16, F32, Layer, check_scan, elt_dtype, from_type, scan, to_type
from nextsycl_amd import DevBuf, Gpu
from nextsycl_amd.attn import Ops

pytestmark = pytest.mark.gpu
E = {F32: 4, F16: 2, BF16: 2}


class Call:
    """A prompt of T rows from position 0 on, x B C and the step sizes in one row, on buffers of its own."""

    def __init__(self, ops, L, qt, raw):
        self.ops, self.L, self.qt, self.T = ops, L, qt, raw.shape[0]
        g, of = ops.gpu, lambda a: None if a is None else DevBuf.of(ops.gpu, a)  # noqa: E731
        self.w = tuple(of(a) for a in (L.cw, L.cb, L.a, L.dtb, L.d))
        self.rows, self.ring = of(raw), of(np.full((4, L.chan), np.nan, np.float32))
        self.y, self.h = DevBuf(g, self.T * L.inner * E[qt]), DevBuf(g, L.H * L.P * L.N * 4)
        self.sc = DevBuf(g, max(4, 4 * ops.ssm_prompt_scratch(self.T, L.H, L.P, L.N, L.G, L.K)))

    def run(self, in_place=False):
        L, e, row = self.L, E[self.qt], self.L.chan + self.L.H
        self.ops.ssm_prompt(self.qt, self.rows, row, self.rows.view(L.chan * e, self.rows.len - L.chan * e), row, *self.w, self.ring, 4, 0, self.T, L.H, L.P, L.N, L.G,
                            L.K, self.h if in_place else None, self.h, self.y, L.inner, self.sc)

    def out(self):
        return from_type(self.qt, self.y.read(elt_dtype(self.qt)).reshape(self.T, -1)), self.h.read(np.float32).reshape(self.L.H, self.L.P, self.L.N)

    def bits(self):
        return self.y.read(np.uint8), self.h.read(np.uint8), self.ring.read(np.uint8)


def rows_of(L, qt, T, seed):
    raw, val = to_type(qt, np.random.default_rng(seed).standard_normal((T, L.chan + L.H)))
    return raw, val


def plain(L, val):
    return scan(L, val[:, :L.chan], val[:, L.chan:], np.zeros((L.K - 1, L.chan)), np.zeros((L.H, L.P, L.N)))


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N,G,K,T,p0,cap", [(4, 64, 128, 2, 4, 1, 0, 4), (4, 64, 128, 2, 4, 16, 3, 19), (2, 50, 100, 1, 4, 9, 2, 40), (3, 8, 33, 3, 3, 5, 50, 7), (2, 16, 256, 1, 1, 12, 9, 1),
                                                (2, 40, 20, 1, 2, 2, 0, 3), (2, 64, 128, 1, 4, 16, 3, 18), (2, 64, 128, 1, 4, 17, 3, 20)])
def test_a_prompt_of_a_few_rows(ops, qt, H, P, N, G, K, T, p0, cap):
    """Those that run row by row and their neighbours: y, the state (h0 kept), and of the rows the last K - 1 in the ring, nothing else."""
    g, e = ops.gpu, E[qt]
    L = Layer(H, P, N, G, K, seed=T)
    raw, val = rows_of(L, qt, T, 14)
    r = np.random.default_rng(15)
    past = r.standard_normal((K - 1, L.chan)).astype(np.float32)
    ring = np.full((cap, L.chan), np.nan, np.float32)
    for k in range(K - 1):
        if p0 - (K - 1) + k < 0:
            past[k] = 0.0
        else:
            ring[(p0 - (K - 1) + k) % cap] = past[k]
    h0 = r.standard_normal((H, P, N)).astype(np.float32)
    y, h, yb, hb = scan(L, val[:, :L.chan], val[:, L.chan:], past, h0)
    c = Call(ops, L, qt, raw)
    ringb, h0b, row = DevBuf.of(g, ring), DevBuf.of(g, h0), L.chan + H
    ops.ssm_prompt(qt, c.rows, row, c.rows.view(L.chan * e, c.rows.len - L.chan * e), row, *c.w, ringb if K > 1 else None, cap, p0, T, H, P, N, G, K, h0b, c.h, c.y, L.inner, c.sc)
    got, state = c.out()
    check_scan(got, y, yb, qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")
    assert np.array_equal(h0b.read(np.float32), h0.ravel())
    for t in range(max(0, T - (K - 1)), T):
        ring[(p0 + t) % cap] = val[t, :L.chan]
    assert np.array_equal(ringb.read(np.uint32), ring.view(np.uint32).ravel())


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("part", ["x", "B", "C", "step"])
@pytest.mark.parametrize("qt,T,at", [(F32, 150, 70), (F32, 600, 333), (BF16, 150, 64), (F16, 600, 63)])
def test_what_is_not_finite_stays_where_the_recurrence_takes_it(ops, qt, T, at, part, bad):
    """One value of a row that is not finite: of x its column from that row on, of B its group's heads (one feature of their
    states), of a step size its head, of C its group's heads in the rows whose convolution holds it - and everything else as
    if it were not there."""
    H, P, N, G, K = 4, 40, 64, 2, 4
    L = Layer(H, P, N, G, K, seed=2)
    raw, val = rows_of(L, qt, T, 3)
    y, h, yb, hb = plain(L, val)
    column = {"x": 1 * P + 7, "B": L.inner + 1 * N + 5, "C": L.inner + (G + 1) * N + 9, "step": L.chan + 2}[part]
    spoilt = val.copy()
    spoilt[at, column] = bad
    c = Call(ops, L, qt, to_type(qt, spoilt)[0])
    c.run()
    got, state = c.out()
    lost, lost_h = np.zeros((T, H, P), bool), np.zeros((H, P, N), bool)
    if part == "x":
        lost[at:, 1, 7], lost_h[1, 7] = True, True
    elif part == "B":
        lost[at:, 2:], lost_h[2:, :, 5] = True, True         # (of the state that feature alone)
    elif part == "C":
        lost[at:at + K, 2:] = True
    elif bad > 0 or np.isnan(bad):
        lost[at:, 2], lost_h[2] = True, True
    else:
        # (a step of nothing: the row leaves the state as it was)
        val = val.copy()
        val[at, column] = -1e30 if qt != F16 else -60000.0
        y, h, yb, hb = plain(L, val)
    lost = lost.reshape(T, -1)
    if part == "C" and not np.isnan(bad):
        # (silu of -inf is taken as it is computed, NaN: a tap's sign says which; either way no number)
        assert not np.isfinite(got[at][lost[at]]).any()
    elif lost.any():
        assert not np.isfinite(got[lost]).any()
    fine = ~lost.any(0)
    check_scan(got[:at], y[:at], yb[:at], qt, T, N, "rows in front")
    if fine.any():
        check_scan(got[:, fine], y[:, fine], yb[:, fine], qt, T, N, "other columns")
    if part == "C":
        check_scan(got[at + K:], y[at + K:], yb[at + K:], qt, T, N, "rows behind")
    if lost_h.any():
        assert not np.isfinite(state[lost_h]).any()
    check_scan(state[~lost_h], h[T][~lost_h], hb[T][~lost_h], F32, T, N, "state")


def test_a_wide_range_of_values_in_a_column(ops):
    """Rows 10^4 times the others, and decays that leave nothing of them a few rows on: those others keep their bits (an operand
    holds 22 bits of a value down to 2^-16 of its column's largest, and 2^-38 of that largest below)."""
    H, P, N, G, K, T = 2, 64, 64, 1, 4, 200
    L = Layer(H, P, N, G, K, seed=4, rate=-3000.0)
    L.dtb[:] = 0.0
    raw, val = rows_of(L, F32, T, 5)
    for t in (0, 9, 40, 64, 65, 130, 190):
        raw[t, :L.chan] *= 1e4
    y, h, yb, hb = plain(L, raw)
    c = Call(ops, L, F32, raw)
    c.run()
    got, state = c.out()
    assert np.isfinite(got).all()
    # (a row's own bound: its sums of absolute values, for each x, B and C an operand's floor beside it - 10^4 of its own size
    # times 2^-38, 2^-24 in all)
    check_scan(got, y, yb, F32, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N,G,T", [(3, 100, 200, 1, 1500), (12, 64, 128, 3, 1000), (1, 16, 256, 1, 4100), (2, 8, 16, 2, 16500)])
def test_long_prompts_in_segments_and_passes(ops, qt, H, P, N, G, T):
    L = Layer(H, P, N, G, 4, seed=T, rate=-0.3)
    raw, val = rows_of(L, qt, T, 6)
    y, h, yb, hb = plain(L, val)
    c = Call(ops, L, qt, raw)
    c.run()
    got, state = c.out()
    check_scan(got, y, yb, qt, T, N, "y")
    check_scan(state, h[T], hb[T], F32, T, N, "state")
    want = np.full((4, L.chan), np.nan, np.float32)
    for t in range(T - 3, T):
        want[t % 4] = val[t, :L.chan]
    assert np.array_equal(c.ring.read(np.uint32), want.view(np.uint32).ravel())


@pytest.mark.parametrize("qt,T", [(F32, 1100), (BF16, 8200), (F16, 130)])
def test_a_prompt_in_a_graph(qt, T):
    """Segments, passes: recorded once, replayed on other rows with eager calls and waits between, each replay the eager call's bits."""
    g = Gpu.open(0)
    ops = Ops(g)
    try:
        L = Layer(4, 32, 64, 2, 4, seed=7)
        c = Call(ops, L, qt, rows_of(L, qt, T, 0)[0])
        start = np.random.default_rng(8).standard_normal(c.h.len // 4).astype(np.float32)

        def reset(rep):
            c.rows.write(rows_of(L, qt, T, 20 + rep)[0])
            c.h.write(start)
            c.ring.write(np.full((4, L.chan), np.nan, np.float32))
            c.y.fill(0xFF)
            c.sc.fill(0xFF)
            g.sync()

        h = C.c_void_p()
        ops.ok(ops.k.q35_graph_begin(ops.raw(), C.byref(h)), "graph begin")
        try:
            c.run(in_place=True)
        finally:
            ops.ok(ops.k.q35_graph_end(ops.raw(), h), "graph end")
        for rep in range(4):
            reset(rep)
            ops.ok(ops.k.q35_graph_launch(ops.raw(), h), "graph launch")
            got = c.bits()
            reset(rep)
            c.run(in_place=True)
            assert all(np.array_equal(a, b) for a, b in zip(got, c.bits())), rep
        ops.k.q35_graph_free(h)
    finally:
        g.close()


def test_two_prompts_at_once(ops):
    """On two handles' streams, each with buffers of its own, unsynchronized: the bits of each alone."""
    other = Gpu.open(0)
    try:
        L = Layer(8, 64, 128, 2, 4, seed=9)
        calls = [Call(o, L, qt, rows_of(L, qt, 1000, i)[0]) for i, (o, qt) in enumerate(((ops, BF16), (Ops(other), F32)))]
        alone = []
        for c in calls:
            c.run()
            c.ops.gpu.sync()
            alone.append(c.bits())
        for _ in range(3):
            for c in calls:
                c.run()
                c.run()
        for c, want in zip(calls, alone):
            c.ops.gpu.sync()
            assert all(np.array_equal(a, b) for a, b in zip(c.bits(), want))
        del calls, c
    finally:
        other.close()


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N", [(4, 80, 128), (2, 50, 100), (2, 16, 16), (16, 64, 128), (16, 80, 128), (20, 90, 124)])
def test_a_verify_passes_rows_are_their_tokens(ops, qt, H, P, N):
    """Seven successive rows of a slot in one call, among another slot's, against seven calls of a row: the same bits."""
    g, R, cap, e = ops.gpu, 7, 16, E[qt]
    L = Layer(H, P, N, 1, 4, seed=11)
    raw, _ = rows_of(L, qt, 2 * R, 12)
    row, of = L.chan + L.H, lambda a: DevBuf.of(g, a)  # noqa: E731
    w, rows = tuple(of(a) for a in (L.cw, L.cb, L.a, L.dtb, L.d)), of(raw)
    r = np.random.default_rng(13)
    h0, ring0 = r.standard_normal((2, H, P, N)).astype(np.float32), r.standard_normal((2, cap, L.chan)).astype(np.float32)
    slots, pos = np.array([0, 1] * R, np.int32), np.repeat(np.arange(R, dtype=np.int32), 2) + np.array([40, 7] * R, np.int32)
    out = []
    for n in (2 * R, 2):
        h, ring, y = of(h0), of(ring0), DevBuf(g, 2 * R * L.inner * e)
        for t in range(0, 2 * R, n):
            at = lambda o: rows.view((t * row + o) * e, rows.len - (t * row + o) * e)  # noqa: E731,B023
            ops.ssm_step(qt, at(0), row, at(L.chan), row, *w, ring, cap, 0, n, H, P, N, 1, 4, h, h, y.view(t * L.inner * e, n * L.inner * e), L.inner, nslots=2,
                         slots=of(slots[t:t + n]), pos=of(pos[t:t + n]))
            g.sync()
        out.append((y.read(np.uint8), h.read(np.uint8), ring.read(np.uint8)))
    assert all(np.array_equal(a, b) for a, b in zip(*out))
