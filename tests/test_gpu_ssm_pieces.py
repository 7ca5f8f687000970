"""ns_ssm_prompt cut into segments whose states are found in pieces - whole ones, shorter last ones, empty ones -, at every width of column tiles and
of states; and half rows, held to operands of 22 bits."""
import types

import numpy as np
import pytest

from layer_ref import BF16, F16, F32, ROUND, TINY, Layer, check_scan, elt_dtype, from_type, scan, scan_tolerance, to_type
from nextsycl_amd import DevBuf
from test_gpu_ssm_edges import E, Call, plain, rows_of

pytestmark = pytest.mark.gpu


def cut(qt, T, H, P, N):
    """How a pass of T rows is cut, by the library's rule: (chunks, segments, chunks a segment, pieces a segment, chunks a piece, column tiles)."""
    wgs = 1 if N > 128 else 3 if qt == BF16 else 2
    chunks, blocks = -(-T // 64), -(-P // 64)
    owners = H * blocks
    segs = max(1, min(32, 256 * wgs // owners, 1 if chunks < 6 else chunks // 2))
    per = -(-chunks // segs)
    segs = -(-chunks // per)
    sub = 1 if segs == 1 else max(1, min(per // 4, -(-768 // (owners * (segs - 1)))))
    tiles = -(--(-P // 16) // blocks)
    return chunks, segs, per, sub, -(-per // sub), max(2, tiles)


def some(L, heads, columns):
    """The layer of a few of its heads and columns alone, each head with its group's B and C: (layer, its channels)."""
    per, x = L.H // L.G, [h * L.P + c for h in heads for c in columns]
    group = lambda o: [L.inner + (o * L.G + h // per) * L.N + n for h in heads for n in range(L.N)]  # noqa: E731
    ch = np.array(x + group(0) + group(1))
    n = len(heads)
    return types.SimpleNamespace(H=n, P=len(columns), N=L.N, G=n, K=L.K, inner=len(x), chan=len(ch), cw=L.cw[ch], cb=L.cb[ch], a=L.a[heads], dtb=L.dtb[heads], d=L.d[heads]), ch


def near_halves(got, ref, what):
    """Half values are the exact ones' roundings, but for those that lie as near a border as 32-bit arithmetic errs: 2^-18 of them in the mean against
    borders 2^-11 of a value apart and more, less for small values among large (6 times: a normal distribution's mean of 1 / size down to 2^-7): 1 in
    16 at most. (Operands of 11 bits would put a third of them beside.)"""
    want = from_type(F16, to_type(F16, ref)[0]).reshape(ref.shape)
    off = (got != want).mean()
    assert off <= 1.0 / 16, "%s: %.3f" % (what, off)


# H, P, N, G, T; (KT, column tiles), whether a piece is empty
CASES = [
    (128, 60, 120, 2, 2790, (2, 4), False), (80, 64, 64, 1, 4129, (1, 4), False), (96, 40, 100, 2, 4100, (2, 3), False), (128, 20, 70, 1, 2801, (2, 2), False),
    (86, 36, 130, 2, 3126, (4, 3), True), (40, 17, 256, 4, 3100, (4, 2), False), (96, 8, 20, 3, 8192 + 4100, (1, 2), False), (12, 200, 140, 2, 2900, (4, 4), False),
]


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,N,G,T,form,empty", CASES)
def test_segments_in_pieces(ops, qt, H, P, N, G, T, form, empty):
    chunks, segs, per, sub, piece, tiles = cut(qt, min(T, 8192), H, P, N)
    assert segs > 1 and sub > 1 and (1 if N <= 64 else 2 if N <= 128 else 4, tiles) == form
    assert ((sub - 1) * piece >= per) == empty
    L = Layer(H, P, N, G, 4, seed=H + P, rate=None)
    L.a *= np.float32(0.02)                        # (a row is felt some thousand rows on: by the segments behind its own)
    raw, val = rows_of(L, qt, T, 51)
    heads, columns = np.array([0, 1, H // 2, H - 2, H - 1]), sorted({0, P // 3, P // 2 + 1, P - 1})
    S, ch = some(L, heads, columns)
    r = np.random.default_rng(52)
    h0 = r.standard_normal((H, P, N)).astype(np.float32)
    at = np.ix_(heads, columns)
    y, h, yb, hb = scan(S, val[:, ch], val[:, L.chan + heads], np.zeros((3, len(ch))), h0[at])
    c = Call(ops, L, qt, raw)
    g, e, row = ops.gpu, E[qt], L.chan + H
    sc = DevBuf(g, c.sc.len + 4096)
    sc.fill(0xFF)
    for in_place in (False, True):
        c.h.write(h0)
        h1 = c.h if in_place else DevBuf(g, c.h.len)
        ops.ssm_prompt(qt, c.rows, row, c.rows.view(L.chan * e, c.rows.len - L.chan * e), row, *c.w, c.ring, 4, 0, T, H, P, N, G, 4, c.h, h1, c.y, L.inner, sc.view(0, c.sc.len))
        got = from_type(qt, c.y.read(elt_dtype(qt)).reshape(T, -1))
        state = h1.read(np.float32).reshape(H, P, N)
        assert np.isfinite(got).all() and np.isfinite(state).all()
        mine = got[:, ch[:S.inner]]
        check_scan(mine, y, yb, qt, T, N, "y")
        if qt != BF16:
            err, tol = np.abs(mine - y), scan_tolerance(T, N) * yb + ROUND[qt] * np.abs(y) + TINY[qt]
            assert (err <= tol).all(), (err / tol).max()
        if qt == F16:
            near_halves(mine, y, "y")
        check_scan(state[at], h[T], hb[T], F32, T, N, "state")
    assert (sc.read(np.uint8, 4096, sc.len - 4096) == 0xFF).all()


@pytest.mark.parametrize("H,P,N,G,T", [(4, 64, 128, 2, 150), (3, 80, 128, 1, 300), (2, 50, 100, 1, 77), (2, 16, 256, 1, 700), (8, 32, 40, 2, 513), (4, 64, 128, 2, 12)])
def test_half_rows_keep_22_bits(ops, H, P, N, G, T):
    L = Layer(H, P, N, G, 4, seed=61)
    raw, val = rows_of(L, F16, T, 62)
    y, h, yb, hb = plain(L, val)
    c = Call(ops, L, F16, raw)
    c.run()
    got, state = c.out()
    near_halves(got, y, "prompt")
    g, row = ops.gpu, L.chan + H
    st, ring, out = DevBuf.of(g, np.zeros((H, P, N), np.float32)), DevBuf.of(g, np.full((4, L.chan), np.nan, np.float32)), DevBuf(g, T * L.inner * 2)
    for t in range(T):
        at = lambda o: c.rows.view((t * row + o) * 2, c.rows.len - (t * row + o) * 2)  # noqa: E731,B023
        ops.ssm_step(F16, at(0), row, at(L.chan), row, *c.w, ring, 4, t, 1, H, P, N, G, 4, st, st, out.view(t * L.inner * 2, L.inner * 2), L.inner)
    near_halves(from_type(F16, out.read(np.uint16).reshape(T, -1)), y, "steps")
