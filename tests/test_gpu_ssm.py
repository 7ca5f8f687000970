"""The state-space mixer - ns_ssm_prompt, ns_ssm_step - against its definition row by row in float64 (layer_ref.py says how
far float32 arithmetic may be from it)."""
import numpy as np
import pytest

from layer_ref import BF16, F16, F32, Layer, check_scan, elt_dtype, from_type, scan, to_type
from nextsycl_amd import DevBuf, Error

pytestmark = pytest.mark.gpu
E = {F32: 4, F16: 2, BF16: 2}


class Weights:
    def __init__(self, g, L):
        opt = lambda a: None if a is None else DevBuf.of(g, a)  # noqa: E731
        self.cw, self.cb, self.a, self.dtb, self.d = DevBuf.of(g, L.cw), opt(L.cb), DevBuf.of(g, L.a), opt(L.dtb), opt(L.d)

    def args(self):
        return self.cw, self.cb, self.a, self.dtb, self.d


def projected(L, qt, T, seed, pad=0, sigma=1.0):
    """Rows [pad | x B C | step sizes | pad] of an in-projection: (raw for the GPU, x B C, step sizes as float32)."""
    r = np.random.default_rng(seed)
    raw, val = to_type(qt, r.standard_normal((T, pad + L.chan + L.H + pad)) * sigma)
    return raw, val[:, pad:pad + L.chan], val[:, pad + L.chan:pad + L.chan + L.H]


def ring_of(L, cap, p0, past):
    """A ring whose slots are NaN but for the rows in front of p0 (those that there are)."""
    ring = np.full((cap, L.chan), np.nan, np.float32)
    for k in range(L.K - 1):
        p = p0 - (L.K - 1) + k
        if p >= 0:
            ring[p % cap] = past[k]
    return ring


def history(L, p0, seed):
    past = np.random.default_rng(seed).standard_normal((L.K - 1, L.chan)).astype(np.float32)
    for k in range(L.K - 1):
        if p0 - (L.K - 1) + k < 0:
            past[k] = 0.0
    return past


# H, P, N, G, K, T, p0, cap, pad
PROMPTS = [
    (2, 64, 128, 1, 4, 64, 0, 4, 0), (2, 64, 128, 1, 4, 1, 0, 3, 0), (4, 64, 128, 2, 4, 65, 7, 4, 8), (2, 64, 128, 2, 4, 200, 1, 5, 16),
    (3, 80, 128, 1, 4, 130, 2, 8, 0), (2, 50, 100, 1, 4, 77, 3, 4, 3), (1, 1, 1, 1, 4, 5, 0, 4, 1), (4, 5, 16, 2, 3, 63, 9, 2, 1),
    (2, 128, 64, 1, 2, 129, 100, 1, 0), (2, 32, 256, 1, 4, 70, 12345678901, 3, 4), (6, 16, 32, 3, 1, 40, 0, 1, 2), (2, 64, 128, 1, 4, 2, 1, 3, 0),
    (2, 64, 128, 1, 4, 3, 50, 7, 0), (1, 200, 130, 1, 4, 66, 5, 4, 2), (8, 8, 8, 8, 4, 300, 0, 4, 8), (16, 64, 128, 1, 4, 513, 0, 4, 8),
]


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N,G,K,T,p0,cap,pad", PROMPTS)
def test_prompt(ops, qt, H, P, N, G, K, T, p0, cap, pad):
    g = ops.gpu
    L = Layer(H, P, N, G, K, seed=H + P + T)
    raw, xbc, step = projected(L, qt, T, seed=T, pad=pad)
    row, e = raw.shape[1], E[qt]
    past = history(L, p0, 5)
    h0 = np.random.default_rng(6).standard_normal((H, P, N)).astype(np.float32) * 0.3
    ring = ring_of(L, cap, p0, past)
    y, h, yb, hb = scan(L, xbc, step, past, h0)
    W = Weights(g, L)
    rows, ringb, h0b = DevBuf.of(g, raw), DevBuf.of(g, ring), DevBuf.of(g, h0)
    ys = L.inner + 3
    yb_, h1b = DevBuf(g, (T + 1) * ys * e), DevBuf(g, h0.nbytes)
    sc = DevBuf(g, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, K) + 64)
    for b in (yb_, sc, h1b):
        b.fill(0xFF)
    at = lambda o: rows.view(o * e, rows.len - o * e)  # noqa: E731
    ops.ssm_prompt(qt, at(pad), row, at(pad + L.chan), row, *W.args(), ringb if K > 1 else None, cap, p0, T, H, P, N, G, K, h0b, h1b, yb_, ys,
                   sc.view(0, sc.len - 64))
    got = yb_.read(elt_dtype(qt)).reshape(T + 1, ys)
    what = "prompt %s" % ((H, P, N, G, K, T, p0),)
    check_scan(from_type(qt, np.ascontiguousarray(got[:T, :L.inner])), y, yb, qt, T, N, what)
    check_scan(h1b.read(np.float32).reshape(h0.shape), h[T], hb[T], F32, T, N, what + " state")
    # nothing beside the rows, behind the last or behind the scratch is written
    ones = np.array(-1).astype(elt_dtype(qt)) if qt else np.uint32(0xFFFFFFFF)
    bits = got.view(np.uint32) if qt == F32 else got
    assert (bits[:T, L.inner:] == ones).all() and (bits[T] == ones).all() and (sc.read(np.uint8, 64, sc.len - 64) == 0xFF).all()
    # the ring: the last K - 1 rows where their positions put them, nothing else changed
    want = ring.copy()
    for t in range(max(0, T - (K - 1)), T):
        want[(p0 + t) % cap] = xbc[t]
    assert np.array_equal(ringb.read(np.uint32), want.view(np.uint32).ravel())
    # in place, and again: the same bits
    if K == 1 or T >= 1:
        ringb.write(ring)
        y2 = DevBuf(g, yb_.len)
        ops.ssm_prompt(qt, at(pad), row, at(pad + L.chan), row, *W.args(), ringb if K > 1 else None, cap, p0, T, H, P, N, G, K, h0b, h0b, y2, ys, sc)
        assert np.array_equal(y2.read(elt_dtype(qt)).reshape(T + 1, ys)[:T, :L.inner].view(bits.dtype), bits[:T, :L.inner])
        assert np.array_equal(h0b.read(np.uint32), h1b.read(np.uint32))


@pytest.mark.parametrize("bias,rate,lo,hi,sigma", [(False, None, 0.0, np.inf, 1.0), (True, -40.0, 0.5, np.inf, 1.0), (True, -1e-4, 0.0, np.inf, 1.0),
                                                   (True, None, 0.02, 0.05, 1.0), (True, -1.0, 0.0, np.inf, 300.0), (True, -1.0, 0.0, np.inf, 1e-4),
                                                   (True, 0.0, 0.0, np.inf, 1.0), (True, -2000.0, 0.5, np.inf, 1.0)])
def test_prompt_rates_limits_and_sizes_of_values(ops, bias, rate, lo, hi, sigma):
    """No biases; decays that leave nothing of a row behind it, and next to none; limited step sizes; large and small rows."""
    g = ops.gpu
    H, P, N, G, K, T = 4, 64, 128, 2, 4, 150
    L = Layer(H, P, N, G, K, seed=3, bias=bias, rate=rate)
    raw, xbc, step = projected(L, F32, T, seed=9, sigma=sigma)
    if sigma != 1.0:
        raw[:, L.chan:] /= sigma
        step = raw[:, L.chan:]
    past = history(L, 0, 1)
    y, h, yb, hb = scan(L, xbc, step, past, np.zeros((H, P, N)), lo, hi)
    W = Weights(g, L)
    rows, ring = DevBuf.of(g, raw), DevBuf.of(g, np.full((4, L.chan), np.nan, np.float32))
    yo, h1, sc = DevBuf(g, T * L.inner * 4), DevBuf(g, H * P * N * 4), DevBuf(g, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, K))
    ops.ssm_prompt(F32, rows, raw.shape[1], rows.view(L.chan * 4, rows.len - L.chan * 4), raw.shape[1], *W.args(), ring, 4, 0, T, H, P, N, G, K, None, h1, yo,
                   L.inner, sc, dt_lo=lo, dt_hi=hi)
    check_scan(yo.read(np.float32).reshape(T, -1), y, yb, F32, T, N, "y")
    check_scan(h1.read(np.float32).reshape(H, P, N), h[T], hb[T], F32, T, N, "state")


def test_prompt_in_pieces_is_the_prompt(ops):
    """A long prompt - more rows than the library works on at a time - whole, and cut where a user would not: the same scan."""
    g = ops.gpu
    H, P, N, G, K, T = 2, 8, 16, 1, 4, 8300
    L = Layer(H, P, N, G, K, seed=1, rate=-0.5)
    raw, xbc, step = projected(L, F32, T, seed=2)
    y, h, yb, hb = scan(L, xbc, step, history(L, 0, 0), np.zeros((H, P, N)))
    W, row = Weights(g, L), raw.shape[1]
    rows, sc = DevBuf.of(g, raw), DevBuf(g, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, K))
    for cuts in ((0, T), (0, 1, 2, 64, 65, 8192, 8193, T)):
        yo, h1, ring = DevBuf(g, T * L.inner * 4), DevBuf(g, H * P * N * 4), DevBuf.of(g, np.full((4, L.chan), np.nan, np.float32))
        for s, e in zip(cuts, cuts[1:]):
            at = lambda o: rows.view((s * row + o) * 4, ((e - s) * row - o) * 4)  # noqa: E731,B023
            ops.ssm_prompt(F32, at(0), row, at(L.chan), row, *W.args(), ring, 4, s, e - s, H, P, N, G, K, h1 if s else None, h1,
                           yo.view(s * L.inner * 4, (e - s) * L.inner * 4), L.inner, sc)
        check_scan(yo.read(np.float32).reshape(T, -1), y, yb, F32, T, N, "y %s" % (cuts,))
        check_scan(h1.read(np.float32).reshape(H, P, N), h[T], hb[T], F32, T, N, "state %s" % (cuts,))


# H, P, N, G, K, slots of the rows, cap
STEPS = [
    (4, 64, 128, 1, 4, [0], 4), (8, 64, 128, 2, 4, [3, 1, 0], 4), (2, 80, 128, 1, 4, [2, 2, 2, 2], 7), (3, 50, 100, 1, 4, [1, 0, 1, 4, 1], 8),
    (2, 64, 16, 2, 3, [5, -1, 7, 2, 100], 3), (2, 20, 64, 1, 2, [0, 1], 2), (4, 64, 256, 4, 4, [1], 9), (2, 9, 30, 1, 1, [0, 0, 3], 1),
    (1, 1, 1, 1, 4, [0], 4), (2, 128, 130, 1, 4, [1, 1], 5), (2, 3, 5, 1, 4, [0, 1, 0, 1, 0, 1, 0, 1], 7), (2, 64, 32, 1, 4, list(range(70)) + [3, 3], 6),
]


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N,G,K,slots,cap", STEPS)
def test_step(ops, qt, H, P, N, G, K, slots, cap):
    """Rows of several slots, in any order, several of one slot, slots that are none: states, rings and rows of those that
    take part, and nothing of the others."""
    g = ops.gpu
    R, nslots, e = len(slots), max(8, max(slots) + 1 if max(slots) < 100 else 8), E[qt]
    L = Layer(H, P, N, G, K, seed=R + N)
    raw, xbc, step = projected(L, qt, R, seed=R, pad=1)
    r = np.random.default_rng(4)
    h0 = r.standard_normal((nslots, H, P, N)).astype(np.float32) * 0.3
    pos = np.zeros(R, np.int32)
    first = r.integers(0, 2 ** 31 - 20, nslots)
    first[0], first[1] = 0, 2                        # (a sequence's first token, and its third)
    seen = {}
    ring = np.full((nslots, cap, L.chan), np.nan, np.float32)
    pasts = {}
    for i, s in enumerate(slots):
        if 0 <= s < nslots:
            pos[i] = first[s] + seen.get(s, 0)
            seen[s] = seen.get(s, 0) + 1
            if s not in pasts:
                pasts[s] = history(L, int(first[s]), 100 + s)
                ring[s] = ring_of(L, cap, int(first[s]), pasts[s])
    want_y, want_h = np.full((R, L.inner), np.nan), h0.astype(np.float64) * 0 - 7.0
    bound_y, bound_h = np.zeros((R, L.inner)), np.zeros(h0.shape)
    want_ring = ring.copy()
    most = cap - K + 1 if K > 1 else R
    for s in pasts:
        idx = [i for i in range(R) if slots[i] == s][:most]
        y, h, yb, hb = scan(L, xbc[idx], step[idx], pasts[s], h0[s])
        want_y[idx], bound_y[idx], want_h[s], bound_h[s] = y, yb, h[-1], hb[-1]
        for j, i in enumerate(idx):
            if K > 1:
                want_ring[s, (int(first[s]) + j) % cap] = xbc[i]
    W, row = Weights(g, L), raw.shape[1]
    rows, ringb = DevBuf.of(g, raw), DevBuf.of(g, ring)
    h0b, h1b = DevBuf.of(g, h0), DevBuf.of(g, np.full(h0.shape, -7.0, np.float32))
    yo = DevBuf(g, R * L.inner * e)
    yo.fill(0xFF)
    ops.ssm_step(qt, rows.view(e, rows.len - e), row, rows.view((1 + L.chan) * e, rows.len - (1 + L.chan) * e), row, *W.args(), ringb if K > 1 else None, cap, 0, R,
                 H, P, N, G, K, h0b, h1b, yo, L.inner, nslots=nslots, slots=DevBuf.of(g, np.array(slots, np.int32)), pos=DevBuf.of(g, pos))
    got = yo.read(elt_dtype(qt)).reshape(R, -1)
    run = ~np.isnan(want_y[:, 0])
    left = got[~run].view(np.uint32) if qt == F32 else got[~run]
    assert (left == (0xFFFFFFFF if qt == F32 else 0xFFFF)).all()
    T = max(seen.values())
    check_scan(from_type(qt, np.ascontiguousarray(got[run])), want_y[run], bound_y[run], qt, T, N, "y")
    check_scan(h1b.read(np.float32).reshape(h0.shape), want_h, bound_h, F32, T, N, "states")
    if K > 1:
        assert np.array_equal(ringb.read(np.uint32), want_ring.view(np.uint32).ravel())
    assert np.array_equal(h0b.read(np.float32), h0.ravel())


def test_steps_follow_a_prompt(ops):
    """A prompt, then its next tokens one at a time in place, slots null and positions counted by the caller, then a verify
    pass whose drafts are not taken and the tokens that come instead: one scan, row by row."""
    g = ops.gpu
    H, P, N, G, K, T, cap = 4, 64, 128, 2, 4, 90, 8
    L = Layer(H, P, N, G, K, seed=8)
    raw, xbc, step = projected(L, F32, T, seed=1)
    y, h, yb, hb = scan(L, xbc, step, history(L, 0, 0), np.zeros((H, P, N)))
    W, row = Weights(g, L), raw.shape[1]
    rows, ring = DevBuf.of(g, raw), DevBuf.of(g, np.full((cap, L.chan), np.nan, np.float32))
    yo, st, spare = DevBuf(g, T * L.inner * 4), DevBuf(g, H * P * N * 4), DevBuf(g, H * P * N * 4)
    sc = DevBuf(g, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, K))
    at = lambda t, o: rows.view((t * row + o) * 4, rows.len - (t * row + o) * 4)  # noqa: E731
    out = lambda t: yo.view(t * L.inner * 4, yo.len - t * L.inner * 4)  # noqa: E731
    ops.ssm_prompt(F32, at(0, 0), row, at(0, L.chan), row, *W.args(), ring, cap, 0, 70, H, P, N, G, K, None, st, out(0), L.inner, sc)
    for t in range(70, 80):
        ops.ssm_step(F32, at(t, 0), row, at(t, L.chan), row, *W.args(), ring, cap, t, 1, H, P, N, G, K, st, st, out(t), L.inner)
    drafts = DevBuf.of(g, np.random.default_rng(0).standard_normal((4, row)).astype(np.float32))
    same = DevBuf.of(g, np.zeros(4, np.int32))
    ops.ssm_step(F32, drafts, row, drafts.view(L.chan * 4, drafts.len - L.chan * 4), row, *W.args(), ring, cap, 80, 4, H, P, N, G, K, st, spare, out(80), L.inner, slots=same)
    # (the state is the one in front of the drafts, and the ring holds the rows in front of them still)
    for t in range(80, T):
        ops.ssm_step(F32, at(t, 0), row, at(t, L.chan), row, *W.args(), ring, cap, t, 1, H, P, N, G, K, st, st, out(t), L.inner)
    check_scan(yo.read(np.float32).reshape(T, -1), y, yb, F32, T, N, "y")
    check_scan(st.read(np.float32).reshape(H, P, N), h[T], hb[T], F32, T, N, "state")


def test_wrappers_check_their_buffers(ops):
    g = ops.gpu
    L = Layer(2, 8, 16, 1, 4, seed=0)
    W, b = Weights(g, L), DevBuf(g, 1 << 16)
    T, row = 3, L.chan + 2
    own = lambda: DevBuf(g, max(1 << 16, 4 * ops.ssm_prompt_scratch(T, 2, 8, 16, 1, 4)))  # noqa: E731
    buffers = dict(ring=own(), h1=own(), y=own(), sc=own())

    def prompt(**k):
        a = dict(rows=b, qt=F32, **buffers)
        a.update(k)
        ops.ssm_prompt(a["qt"], a["rows"], row, b, row, *W.args(), a["ring"], 4, 0, T, 2, 8, 16, 1, 4, None, a["h1"], a["y"], 16, a["sc"])

    prompt()
    for name, size in (("rows", (T - 1) * row * 4 + L.chan * 4 - 4), ("ring", 4 * L.chan * 4 - 4), ("h1", 2 * 8 * 16 * 4 - 4), ("y", T * 16 * 4 - 4),
                       ("sc", ops.ssm_prompt_scratch(T, 2, 8, 16, 1, 4) * 4 - 4)):
        with pytest.raises(Error, match="needs"):
            prompt(**{name: buffers.get(name, b).view(0, size)})
    with pytest.raises(Error, match="rows of type"):
        prompt(qt=3)
    g.sync()
