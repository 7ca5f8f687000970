"""Caches of 8-bit values in blocks of tokens (include/ns_kv8.h) on the GPU: stores and evictions bit for bit, attention and
the weights it gives against 64 bits."""
import numpy as np
import pytest

from kv8_ref import BF16, E4M3, F16, F32, INT8, ROUND, Cache, encode, from_type, same_codes, to_type, tolerance, values
from nextsycl_amd import DevBuf
from nextsycl_amd.attn import TUNE_SCRATCH_MIB, Kv8

pytestmark = pytest.mark.gpu


def on_gpu(ops, c):
    b = [DevBuf.of(ops.gpu, x) for x in (c.k, c.v, c.ks, c.vs)]
    return Kv8(c.form, c.blocks, c.Hkv, c.B, c.D, *b)


def back(c, d):
    """The GPU's pools and scales, shaped as the reference's."""
    return (d.k.read(np.uint8).reshape(c.k.shape), d.v.read(np.uint8).reshape(c.v.shape), d.ks.read(np.float32).reshape(c.ks.shape), d.vs.read(np.float32).reshape(c.vs.shape))


def check_pools(c, d, what=""):
    k, v, ks, vs = back(c, d)
    assert np.array_equal(ks, c.ks) and np.array_equal(vs, c.vs), what + " scales"
    assert same_codes(c.form, k, c.k) and same_codes(c.form, v, c.v), what + " codes"


def ints(ops, x):
    return DevBuf.of(ops.gpu, np.asarray(x, np.int32))


def tables(r, S, tmax, blocks):
    return r.permutation(blocks)[:S * tmax].reshape(S, tmax).astype(np.int32)


def rows_of(qt, r, T, Hkv, D, sigma=1.0, pad=0, shift=0):
    """Rows T x Hkv D, `pad` elements between them, the first `shift` elements into the buffer: (GPU array, stride, values)."""
    x = r.standard_normal((T, Hkv, D)) * sigma * np.exp(0.5 * r.standard_normal((1, Hkv, D)))
    raw, val = to_type(qt, x)
    buf = np.zeros(shift + T * (Hkv * D + pad), raw.dtype)
    for t in range(T):
        buf[shift + t * (Hkv * D + pad):][:Hkv * D] = raw[t].ravel()
    return buf, Hkv * D + pad, val


def store(ops, c, d, qt, k, ks, v, vs, T, table, lens, start, most, shift=0):
    e = 4 if qt == F32 else 2
    kb, vb = DevBuf.of(ops.gpu, k), DevBuf.of(ops.gpu, v)
    ops.kv8_store(d, qt, kb.view(shift * e, kb.len - shift * e), ks, vb.view(shift * e, vb.len - shift * e), vs, T, ints(ops, table), table.shape[1], len(lens), most,
                  ints(ops, lens), start=None if start is None else ints(ops, start))
    ops.gpu.sync()


# ---- the store

STORES = [  # D, B, contexts, rows, most
    (128, 64, [0], [1], 1),
    (128, 16, [5, 0, 31], [1, 1, 1], 1),
    (256, 32, [0, 63, 64, 65], [70, 1, 2, 33], 70),
    (128, 128, [200, 0], [0, 300], 300),
    (256, 128, [127, 1], [129, 256], 256),
    (256, 16, [15, 16], [1, 40], 40),
    (128, 32, [3, 40], [9, 50], 20),                       # rows behind a sequence's first 20 are not stored
]


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("D,B,lens,counts,most", STORES)
def test_store(ops, form, qt, D, B, lens, counts, most):
    r = np.random.default_rng(D + B + len(lens))
    Hkv, S = 3, len(lens)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    T, tmax = int(start[-1]), max((a + b + B - 1) // B for a, b in zip(lens, counts)) + 1
    c = Cache(form, S * tmax + 2, Hkv, B, D, seed=B)
    c.k[:], c.v[:] = encode(form, 30 * r.standard_normal(c.k.shape)), encode(form, 30 * r.standard_normal(c.k.shape))   # (re-rounding NaN codes is not asked for)
    d, table = on_gpu(ops, c), tables(r, S, tmax, c.blocks)
    k, ks, kv = rows_of(qt, r, T, Hkv, D, 20.0, pad=5, shift=3)
    v, vs, vv = rows_of(qt, r, T, Hkv, D, 0.01, pad=0, shift=3)
    store(ops, c, d, qt, k, ks, v, vs, T, table, np.array(lens), start, most, shift=3)
    c.store(kv, vv, table, lens, start, most)
    check_pools(c, d)


@pytest.mark.parametrize("form", [INT8, E4M3])
def test_a_token_at_a_time_grows_a_blocks_scale(ops, form):
    """Tokens of growing magnitude one by one: the block's scale doubles, what is there is re-rounded, all as the definition says."""
    r = np.random.default_rng(7)
    Hkv, B, D = 2, 16, 128
    c = Cache(form, 3, Hkv, B, D, seed=1)
    d, table = on_gpu(ops, c), np.array([[2, 0]], np.int32)
    seen = []
    for t in range(20):
        x = r.standard_normal((1, Hkv, D)) * 2.0 ** (t / 2 - 4)
        raw, val = to_type(BF16, x)
        seen.append(val)
        store(ops, c, d, BF16, raw, Hkv * D, raw, Hkv * D, 1, table, np.array([t]), None, 1)
        c.store(val, val, table, [t], [0, 1], 1)
        check_pools(c, d, "token %d" % t)
    # and each stays within a step of its block's final scale (e4m3: and half a step of its own 3 bits, at each rounding)
    k, _ = c.tokens(table, 0, 20)
    for t in range(20):
        s = c.ks[table[0, t // B]].astype(np.float64)[:, None]
        x, most = seen[t][0], c.ks[table[0, t // B]].astype(np.float64)[:, None] * (127 if form == INT8 else 448)
        assert (np.abs(x) <= most).all()
        assert (np.abs(k[t] - x) <= (s if form == INT8 else np.maximum(np.abs(x) / 8, s * 2.0 ** -8))).all()


@pytest.mark.parametrize("form", [INT8, E4M3])
def test_store_values_at_the_ends(ops, form):
    """Zeros, the smallest and largest values, values between two codes, NaN and infinities."""
    D, B = 128, 16
    c = Cache(form, 6, 1, B, D, seed=2)
    d, table = on_gpu(ops, c), np.arange(6, dtype=np.int32)[None]
    top = 127.0 if form == INT8 else 448.0
    x = np.zeros((6 * B, 1, D), np.float32)
    x[B:2 * B] = 1e-38                                                 # a block of next to nothing
    x[2 * B, 0, :4] = [np.inf, -np.inf, 3e38, 1.0]
    x[3 * B, 0, :6] = [np.nan, 5.0, -5.0, 0.3, 1e-30, -0.0]
    x[4 * B, 0, 0] = top * 2.0 ** -3                                   # exactly the largest code
    x[4 * B, 0, 1:D] = (np.arange(1, D) - 0.5) * 2.0 ** -3             # ties
    x[5 * B, 0, 0] = np.nextafter(np.float32(top), np.float32(1e9))    # just past it: the next scale
    x[5 * B, 0, 1:D] = np.arange(1, D)
    store(ops, c, d, F32, x.reshape(-1, D), D, x.reshape(-1, D), D, len(x), table, np.array([0]), np.array([0, len(x)]), len(x))
    c.store(x.astype(np.float64), x.astype(np.float64), table, [0], [0, len(x)], len(x))
    check_pools(c, d)


def test_store_leaves_what_it_does_not_write(ops):
    """Rows of no sequence, sequences of negative or too large length, entries that are no blocks, positions past the table."""
    r = np.random.default_rng(3)
    Hkv, B, D = 2, 16, 128
    c = Cache(INT8, 9, Hkv, B, D, seed=5)
    d = on_gpu(ops, c)
    table = np.array([[0, -1, 1], [9, 2, 3], [4, 5, 6], [7, 8, -7]], np.int32)
    lens, start = np.array([10, 14, -1, (1 << 30) + 1]), np.array([2, 40, 80, 85, 90])
    k, ks, kv = rows_of(F16, r, 95, Hkv, D)
    store(ops, c, d, F16, k, ks, k, ks, 95, table, lens, start, 64)
    c.store(kv, kv, table, [10, 14, -1, -1], start, 64)
    check_pools(c, d)


# ---- attention

def filled(r, form, blocks, Hkv, B, D, table, lens, seed=0, sigma=1.0):
    """A cache whose sequences' tokens are stored, garbage around them, and float64 copies of nothing: the reference reads the codes."""
    c = Cache(form, blocks, Hkv, B, D, seed)
    for s, n in enumerate(lens):
        if n > 0:
            x = [r.standard_normal((n, Hkv, D)) * sigma * np.exp(0.4 * r.standard_normal((1, Hkv, D))) for _ in range(2)]
            one = np.zeros(len(lens) + 1, int)
            one[s + 1:] = n
            c.store(*x, table, [0 if i == s else -1 for i in range(len(lens))], one, n)
    return c


def attend(ops, c, d, qt, q, qs, table, lens, start, T, most, Hq, longest=None, win=0, scale=0.0, acc0=None, acc1=None, fill=0xFF):
    g = ops.gpu
    longest = longest or max(int(a) + most for a in lens if a < 1 << 30)
    qb, ob = DevBuf.of(g, q), DevBuf(g, T * Hq * c.D * (4 if qt == F32 else 2))
    ob.fill(fill)
    n = ops.kv8_attend_scratch(len(lens), most, Hq, c.Hkv, c.D, longest, acc1 is not None)
    sc = DevBuf(g, max(4, 4 * n))
    sc.fill(0xFF)
    ops.kv8_attend(d, qt, qb, qs, T, ints(ops, table), table.shape[1], len(lens), most, longest, ints(ops, lens), Hq, ob, sc, start=None if start is None else ints(ops, start),
                   win=win, scale=scale, acc0=acc0, acc1=acc1)
    g.sync()
    return ob.read(np.float32 if qt == F32 else np.uint16).reshape(T, Hq, c.D)


def check_rows(qt, raw, ref, q, k, v, D, scale=0.0, what=""):
    got = from_type(qt, raw)
    Hq, Hkv = q.shape[1], k.shape[1]
    reach = max(float((np.abs(q[:, h]) @ np.abs(k[:, h * Hkv // Hq]).T).max()) for h in range(Hq)) * (scale or D ** -0.5) * np.log2(np.e)
    tol, rel = tolerance(qt, ref, reach, float(np.abs(v).max()), D, len(k))
    assert np.isfinite(got).all(), what
    assert np.abs(got - ref).max() <= tol, "%s: %.3g (<= %.3g)" % (what, np.abs(got - ref).max(), tol)
    assert np.linalg.norm(got - ref) <= rel * np.linalg.norm(ref) + 1e-12, "%s: relative L2 %.3g" % (what, np.linalg.norm(got - ref) / np.linalg.norm(ref))


ATTENDS = [  # Hq, Hkv, D, B, contexts, rows each, most, window
    (8, 8, 128, 64, [0], [1], 1, 0),
    (32, 8, 128, 64, [4095], [1], 1, 0),
    (32, 8, 128, 16, [1, 31, 32, 33, 700], [1, 1, 1, 1, 1], 1, 0),
    (24, 4, 256, 128, [1003, 0, 129], [4, 1, 3], 4, 0),
    (64, 4, 128, 32, [3000], [1], 1, 0),
    (5, 1, 128, 64, [517, 64], [16, 7], 16, 0),
    (28, 4, 128, 16, [2100, 90], [2, 16], 16, 100),
    (16, 2, 256, 32, [255, 1500, 40], [5, 2, 1], 5, 64),
    (6, 3, 256, 16, [17], [1], 1, 1),
    (40, 1, 128, 128, [260], [2], 2, 0),
    (3, 3, 128, 32, [130, 5000], [1, 2], 2, 0),
]


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,B,lens,counts,most,win", ATTENDS)
def test_attend(ops, form, qt, Hq, Hkv, D, B, lens, counts, most, win):
    r = np.random.default_rng(Hq + D + B)
    S = len(lens)
    ends = [a + b for a, b in zip(lens, counts)]
    tmax = max((e + B - 1) // B for e in ends)
    table = tables(r, S, tmax, S * tmax + 1)
    c = filled(r, form, S * tmax + 1, Hkv, B, D, table, ends, seed=B)
    d = on_gpu(ops, c)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    T = int(start[-1])
    q, qs, qv = rows_of(qt, r, T, Hq, D, pad=8)
    acc0 = r.uniform(0, 3, (c.blocks, Hkv, B)).astype(np.float32)
    a0, a1 = DevBuf.of(ops.gpu, acc0), DevBuf.of(ops.gpu, np.full_like(acc0, -1))
    raw = attend(ops, c, d, qt, q, qs, table, lens, start, T, most, Hq, win=win, acc0=a0, acc1=a1)
    want = np.full(acc0.shape, -1.0)
    for s in range(S):
        a, b = start[s], start[s + 1]
        ref, given = c.attend(qv[a:b], table, s, lens[s], win)
        k, v = c.tokens(table, s, ends[s])
        check_rows(qt, raw[a:b], ref, qv[a:b], k, v, D, what="sequence %d" % s)
        c.give(acc0.astype(np.float64), want, table, s, lens[s], given)
    got = a1.read(np.float32).reshape(acc0.shape)
    # a weight's relative error as the rows', the sum's roundings
    assert np.abs(got - want).max() <= 2.0 ** -17 * max(1.0, want.max())
    # the same without weights, bit for bit
    again = attend(ops, c, d, qt, q, qs, table, lens, start, T, most, Hq, win=win)
    assert np.array_equal(again, raw)


def test_attend_one_row_each_and_shared_prefixes(ops):
    """start null: sequence s has row s; two sequences whose first blocks are the same ones; sequences without a row."""
    r = np.random.default_rng(11)
    Hq, Hkv, D, B = 8, 2, 128, 32
    table = np.array([[3, 1, 0], [3, 1, 5], [2, 4, 6]], np.int32)
    c = filled(r, E4M3, 8, Hkv, B, D, table, [70, 70, 64])
    # (the second sequence's store went into blocks 3 and 1 last: both read the same)
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(BF16, r, 2, Hq, D)
    raw = attend(ops, c, d, BF16, q, qs, table, np.array([69, 66, 10]), None, 2, 1, Hq)
    for s, n in ((0, 69), (1, 66)):
        ref, _ = c.attend(qv[s:s + 1], table, s, n)
        check_rows(BF16, raw[s:s + 1], ref, qv[s:s + 1], *c.tokens(table, s, n + 1), D)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("B", [16, 64])
def test_attend_entries_that_are_no_blocks(ops, form, B):
    """Their tokens are keys and values of zeros, also past the table's end; nothing is written for them."""
    r = np.random.default_rng(B)
    Hq, Hkv, D, n = 4, 2, 128, 5 * B
    table = np.array([[0, -1, 7, 1 << 30, 2]], np.int32)
    c = filled(r, form, 4, Hkv, B, D, table, [n])
    d = on_gpu(ops, c)
    for qt, cut in ((F32, 5), (F16, 3)):
        t = np.ascontiguousarray(table[:, :cut])
        q, qs, qv = rows_of(qt, r, 2, Hq, D)
        acc = DevBuf.of(ops.gpu, np.full((4, Hkv, B), -1, np.float32))
        raw = attend(ops, c, d, qt, q, qs, t, np.array([n - 2]), np.array([0, 2]), 2, 2, Hq, acc1=acc)
        ref, given = c.attend(qv, t, 0, n - 2)
        check_rows(qt, raw, ref, qv, *c.tokens(t, 0, n), D)
        want = np.full((4, Hkv, B), -1.0)
        c.give(None, want, t, 0, n - 2, given)
        assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17


def test_attend_leaves_other_rows_and_sees_no_further_than_longest(ops):
    r = np.random.default_rng(4)
    Hq, Hkv, D, B = 8, 4, 128, 16
    lens, start = np.array([40, -5, 100, 7]), np.array([1, 3, 5, 6, 9])
    table = tables(r, 4, 8, 40)
    c = filled(r, INT8, 40, Hkv, B, D, table, [42, 0, 101, 10])
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(F32, r, 12, Hq, D)
    raw = attend(ops, c, d, F32, q, qs, table, lens, start, 12, 2, Hq, longest=60, fill=0x11)
    untouched = np.full((Hq, D), 0x11111111, np.uint32)
    for row in (0, 3, 4, 8, 9, 10, 11):               # in front, of the negative one, behind the first two, behind the last
        assert np.array_equal(raw[row].view(np.uint32), untouched), row
    for s in (0, 2, 3):
        a = start[s]
        b = min(start[s + 1], a + 2)
        ref, _ = c.attend(qv[a:b], table, s, lens[s], longest=60)
        check_rows(F32, raw[a:b], ref, qv[a:b], *c.tokens(table, s, int(lens[s]) + b - a), D, what=str(s))


def test_attend_rows_that_see_nothing(ops):
    """`longest` in front of a row's window: zeros."""
    r = np.random.default_rng(5)
    table = np.arange(8, dtype=np.int32)[None]
    c = filled(r, INT8, 8, 1, 16, 128, table, [120])
    q, qs, _ = rows_of(F32, r, 1, 2, 128)
    for longest in (40, 70):
        raw = attend(ops, c, on_gpu(ops, c), F32, q, qs, table, np.array([119]), None, 1, 1, 2, longest=longest, win=30)
        assert not raw.any()


def test_attend_wide_ranges(ops):
    """Rows of very large and very small values, rows of zeros, blocks at both ends of the scales' range, NaN and infinity in one row only."""
    r = np.random.default_rng(6)
    Hq, Hkv, D, B, n = 4, 2, 128, 16, 96
    table = np.arange(6, dtype=np.int32)[None]
    for form in (INT8, E4M3):
        c = filled(r, form, 6, Hkv, B, D, table, [n])
        c.vs[:3], c.vs[3:] = 2.0 ** (-24 if form == INT8 else -15), 2.0 ** (9 if form == INT8 else 7)
        c.ks[2] = 2.0 ** -15
        d = on_gpu(ops, c)
        q, qs, qv = rows_of(F32, r, 6, Hq, D)
        q = q.reshape(6, -1)
        q[1] *= np.float32(1e-30)
        q[2] = 0
        q[3] *= np.float32(40.0)
        q[4, 5], q[5, 5] = np.nan, np.inf
        qv = q.astype(np.float64).reshape(6, Hq, D)
        raw = attend(ops, c, d, F32, q, qs, table, np.array([n - 6]), np.array([0, 6]), 6, 6, Hq)
        assert np.isnan(raw[4:, 0]).all()
        ref, _ = c.attend(qv[:4], table, 0, n - 6)
        k, v = c.tokens(table, 0, n)
        for i in range(4):
            check_rows(F32, raw[i:i + 1], ref[i:i + 1], qv[i:i + 1], k, v, D, what="row %d" % i)
        fine = np.nan_to_num(qv, nan=0.0, posinf=0.0)
        ref, _ = c.attend(fine, table, 0, n - 6)
        check_rows(F32, raw[4:, 2:], ref[4:, 2:], fine[4:, 2:], k[:, 1:], v[:, 1:], D, what="the other key head")
        for i in (4, 5):
            check_rows(F32, raw[i:i + 1, 1:2], ref[i:i + 1, 1:2], fine[i:i + 1, 1:2], k[:, :1], v[:, :1], D, what="the head beside row %d's" % i)


# ---- prompts

PROMPTS = [  # Hq, Hkv, D, B, T, p0, window
    (8, 2, 128, 64, 300, 0, 0),
    (32, 8, 128, 32, 37, 1000, 0),
    (16, 2, 256, 16, 115, 333, 0),
    (24, 4, 256, 128, 20, 5, 0),
    (8, 8, 128, 16, 200, 450, 100),
    (6, 3, 256, 64, 130, 70, 33),
    (8, 4, 128, 64, 5, 200, 0),
    (10, 1, 128, 32, 16, 90, 40),
]


def prompt_close(qt, got, ref, q, k, v, D):
    """A half cache's prompt pass: a query row, scaled, and a weight enter the products as one half each (11 bits: off by at most u = 2^-11 of
    themselves). A score of reach sum |q k| scale moves by up to u times that, a weight by that and u of itself, a mean of values up to vmax by
    twice as much. In the mean the products' roundings add as squares: u sqrt(sum (q k)^2) scale a score, a weight's own u beside it."""
    Hq, Hkv, u = q.shape[1], k.shape[1], 2.0 ** -11
    pairs = [(q[:, h], k[:, h * Hkv // Hq]) for h in range(Hq)]
    reach = max(float((np.abs(a) @ np.abs(b).T).max()) for a, b in pairs) * D ** -0.5
    mean = max(float(np.sqrt((a * a) @ (b * b).T).max()) for a, b in pairs) * D ** -0.5
    assert np.isfinite(got).all()
    assert np.abs(got - ref).max() <= 2 * u * (reach + 1) * np.abs(v).max() + ROUND[qt] * np.abs(ref).max()
    assert np.linalg.norm(got - ref) <= (u * (mean + 1) + ROUND[qt]) * np.linalg.norm(ref)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,B,T,p0,win", PROMPTS)
def test_prompt(ops, form, qt, Hq, Hkv, D, B, T, p0, win):
    r = np.random.default_rng(T + p0)
    tmax = (p0 + T + B - 1) // B
    table = tables(r, 1, tmax, tmax + 2)
    c = filled(r, form, tmax + 2, Hkv, B, D, table, [p0 + T], sigma=0.7)
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(qt, r, T, Hq, D, pad=8)
    ob = DevBuf(ops.gpu, T * Hq * D * (4 if qt == F32 else 2))
    ob.fill(0xFF)
    ops.kv8_prompt(d, qt, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, ob, win=win)
    ops.gpu.sync()
    ref, _ = c.attend(qv, table, 0, p0, win)
    prompt_close(qt, from_type(qt, ob.read(np.float32 if qt == F32 else np.uint16)).reshape(ref.shape), ref, qv, *c.tokens(table, 0, p0 + T), D)


def test_prompt_whose_values_do_not_fit_the_scratch(ops, tune):
    r = np.random.default_rng(8)
    Hq, Hkv, D, B, T, p0 = 8, 4, 128, 32, 70, 900
    tmax = (p0 + T + B - 1) // B
    table = tables(r, 1, tmax, tmax)
    table[0, 3] = -1
    c = filled(r, INT8, tmax, Hkv, B, D, table, [p0 + T], sigma=0.7)
    q, qs, qv = rows_of(F32, r, T, Hq, D)
    ref, _ = c.attend(qv, table, 0, p0)
    outs = []
    for mib in (0, 2, 1):                              # (970 tokens x 4 heads of halfs: 1.9 MiB)
        tune(TUNE_SCRATCH_MIB, mib)
        ob = DevBuf(ops.gpu, T * Hq * D * 4)
        ops.kv8_prompt(on_gpu(ops, c), F32, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, ob)
        ops.gpu.sync()
        outs.append(ob.read(np.float32).reshape(ref.shape))
        prompt_close(F32, outs[-1].astype(np.float64), ref, qv, *c.tokens(table, 0, p0 + T), D)
    check_rows(F32, outs[1], ref, qv, *c.tokens(table, 0, p0 + T), D)      # the rows as a token's: 22 bits


# ---- weights

WEIGHTS = [  # Hq, Hkv, D, B, T, p0, window
    (4, 4, 128, 16, 1, 0, 0),
    (32, 8, 128, 64, 64, 700, 0),
    (24, 4, 256, 32, 50, 301, 0),
    (10, 1, 128, 128, 7, 260, 0),
    (16, 2, 256, 16, 33, 90, 40),
    (8, 2, 128, 32, 300, 0, 0),
    (9, 3, 128, 64, 100, 1500, 200),
    (64, 4, 128, 16, 3, 2500, 0),
    (8, 8, 128, 64, 16, 500, 0),                           # few pairs: as a token's
    (32, 2, 128, 32, 16, 260, 0),
    (48, 1, 256, 64, 9, 700, 90),
    (32, 8, 128, 16, 8, 2100, 300),
    (24, 4, 256, 32, 5, 90, 0),
    (40, 1, 128, 128, 1, 3700, 0),
    (16, 1, 256, 16, 2, 1203, 1),
    (8, 4, 128, 32, 16, 3, 0),
]


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,B,T,p0,win", WEIGHTS)
def test_weights(ops, form, qt, Hq, Hkv, D, B, T, p0, win):
    r = np.random.default_rng(T + p0)
    tmax = (p0 + T + B - 1) // B
    table = tables(r, 1, tmax, tmax + 1)
    if tmax > 4:
        table[0, 2] = -1
    c = filled(r, form, tmax + 1, Hkv, B, D, table, [p0 + T])
    q, qs, qv = rows_of(qt, r, T, Hq, D, pad=3)
    acc0 = r.uniform(0, 3, (c.blocks, Hkv, B)).astype(np.float32)
    want = np.full(acc0.shape, -1.0)
    _, given = c.attend(qv, table, 0, p0, win)
    c.give(acc0.astype(np.float64), want, table, 0, p0, given)
    a1 = DevBuf.of(ops.gpu, np.full_like(acc0, -1))
    ops.kv8_weights(on_gpu(ops, c), qt, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, DevBuf.of(ops.gpu, acc0), a1, win=win)
    ops.gpu.sync()
    got = a1.read(np.float32).reshape(acc0.shape)
    # a weight as the rows' (2^-17 in the mean; here of sums of T G of them), the sum's own roundings
    assert np.abs(got - want).max() <= 2.0 ** -17 * max(1.0, want.max())
    assert np.linalg.norm(got - want) <= 2.0 ** -18 * np.linalg.norm(want)


def test_few_rows_weights_where_the_scratch_holds_no_scores(ops, tune):
    """4 rows of 8 x 2 heads behind 5000 tokens: with 1 MiB the way of many rows; the same sums but for roundings, both into themselves."""
    r = np.random.default_rng(10)
    Hq, Hkv, D, B, T, p0 = 16, 8, 128, 64, 4, 5000
    tmax = (p0 + T + B - 1) // B
    table = tables(r, 1, tmax, tmax)
    c = filled(r, E4M3, tmax, Hkv, B, D, table, [p0 + T])
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(BF16, r, T, Hq, D)
    acc0 = r.uniform(0, 3, (c.blocks, Hkv, B)).astype(np.float32)
    want = acc0.astype(np.float64)
    c.give(want.copy(), want, table, 0, p0, c.attend(qv, table, 0, p0)[1])
    for mib in (0, 1):
        tune(TUNE_SCRATCH_MIB, mib)
        acc = DevBuf.of(ops.gpu, acc0)
        ops.kv8_weights(d, BF16, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, acc, acc)
        ops.gpu.sync()
        assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * want.max(), mib


def test_weights_in_pieces(ops, tune):
    """Rows and heads a few at a time, where the scratch holds no more: the same sums; and without acc0, into itself."""
    r = np.random.default_rng(9)
    Hq, Hkv, D, B, T, p0 = 16, 8, 128, 32, 40, 500
    tmax = (p0 + T + B - 1) // B
    table = tables(r, 1, tmax, tmax)
    c = filled(r, INT8, tmax, Hkv, B, D, table, [p0 + T])
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(F32, r, T, Hq, D)
    want = np.zeros((c.blocks, Hkv, B))
    c.give(None, want, table, 0, p0, c.attend(qv, table, 0, p0)[1])
    for mib in (0, 1):
        tune(TUNE_SCRATCH_MIB, mib)
        acc = DevBuf.of(ops.gpu, np.zeros(want.shape, np.float32))
        ops.kv8_weights(d, F32, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, None, acc)
        ops.gpu.sync()
        got = acc.read(np.float32).reshape(want.shape)
        assert np.abs(got - want).max() <= 2.0 ** -17 * want.max(), mib
    # in two calls, the second on top of the first
    acc = DevBuf.of(ops.gpu, np.full(want.shape, 7, np.float32))
    e = 25 * qs * 4
    qb = DevBuf.of(ops.gpu, q)
    ops.kv8_weights(d, F32, qb, qs, 25, ints(ops, table), tmax, p0, Hq, None, acc)
    ops.kv8_weights(d, F32, qb.view(e, qb.len - e), qs, 15, ints(ops, table), tmax, p0 + 25, Hq, acc, acc)
    ops.gpu.sync()
    got = acc.read(np.float32).reshape(want.shape)
    there = np.zeros(want.shape, bool)
    for t in range(p0 + T):
        there[table[0, t // B], :, t % B] = True
    assert np.abs(got - want)[there].max() <= 2.0 ** -17 * want.max() and (got[~there] == 7).all()


# ---- eviction

EVICTS = [  # Hkv, D, B, contexts, keep, first, last, longest
    (2, 128, 16, [100], 30, 2, 5, 100),
    (3, 256, 32, [500, 77, 130, 0, -3], 100, 1, 31, 500),
    (1, 128, 64, [1000], 999, 0, 0, 1000),
    (2, 128, 128, [700, 300], 64, 32, 32, 700),          # the first and the last ones are all there is room for
    (4, 128, 16, [40, 900], 1, 0, 0, 600),               # one token; a sequence longer than said is passed over
    (2, 256, 16, [333], 200, 4, 0, 4000),
]


def evict_case(r, form, Hkv, D, B, lens, spare=0):
    S = len(lens)
    tmax = max((max(n, 1) + B - 1) // B for n in lens)
    blocks = S * tmax + spare
    table = r.permutation(S * tmax).reshape(S, tmax).astype(np.int32)
    c = Cache(form, blocks, Hkv, B, D, seed=B)
    c.k[:], c.v[:] = encode(form, 40 * r.standard_normal(c.k.shape)), encode(form, 40 * r.standard_normal(c.k.shape))
    acc = np.exp(2 * r.standard_normal((blocks, Hkv, B))).astype(np.float32)
    acc[acc < 0.3] = 0                                   # ties
    acc[acc > 30] = np.inf
    acc[r.random(acc.shape) < 0.02] = np.nan
    acc[r.random(acc.shape) < 0.02] = -1
    return c, table, acc, tmax


def run_evict(ops, c, table, acc, lens, keep, first, last, longest, to=None, alias=False):
    d, ab = on_gpu(ops, c), DevBuf.of(ops.gpu, acc)
    lb = ints(ops, lens)
    l1 = lb if alias else ints(ops, np.full(len(lens), 77))
    ops.kv8_evict(d, ab, ints(ops, table), table.shape[1], len(lens), longest, lb, l1, keep, first, last, to=None if to is None else ints(ops, to))
    ops.gpu.sync()
    return d, ab.read(np.float32).reshape(acc.shape), l1.read(np.int32)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("Hkv,D,B,lens,keep,first,last,longest", EVICTS)
def test_evict_in_place(ops, form, Hkv, D, B, lens, keep, first, last, longest):
    r = np.random.default_rng(B + keep)
    c, table, acc, tmax = evict_case(r, form, Hkv, D, B, lens)
    before = Cache.__new__(Cache)
    before.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()}
    d, got, l1 = run_evict(ops, before, table, acc, lens, keep, first, last, longest, alias=True)
    want = acc.copy()
    new = c.evict(want, table, np.array(lens), keep, first, last, longest=longest)
    assert np.array_equal(l1, new) and np.array_equal(got, want, equal_nan=True)
    # (in the last block of a shortened sequence rows behind its last token count for nothing: compare what is there)
    k, v, ks, vs = back(c, d)
    for s, n in enumerate(new):
        for t in range(max(0, n)):
            b, i = table[s, t // B], t % B
            assert same_codes(form, k[b, :, i], c.k[b, :, i]) and same_codes(form, v[b, :, i], c.v[b, :, i]), (s, t)
            assert np.array_equal(ks[b], c.ks[b]) and np.array_equal(vs[b], c.vs[b]), (s, t)
    check_pools(c, d)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("Hkv,D,B,lens,keep,first,last,longest", EVICTS)
def test_evict_into_fresh_blocks(ops, form, Hkv, D, B, lens, keep, first, last, longest):
    r = np.random.default_rng(B + keep + 1)
    need = (min(keep, max(lens)) + B - 1) // B
    c, table, acc, tmax = evict_case(r, form, Hkv, D, B, lens, spare=len(lens) * need)
    to = np.full(table.shape, -1, np.int32)
    to[:, :need] = table.size + r.permutation(len(lens) * need).reshape(len(lens), need)
    if need > 2:
        to[0, 1] = -9                                    # nothing is written for it
    before = Cache.__new__(Cache)
    before.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()}
    d, got, l1 = run_evict(ops, before, table, acc, lens, keep, first, last, longest, to=to)
    want = acc.copy()
    new = c.evict(want, table, np.array(lens), keep, first, last, to=to, longest=longest)
    assert np.array_equal(l1, new) and np.array_equal(got, want, equal_nan=True)
    check_pools(c, d)


def test_evict_a_long_context_and_equal_weights(ops):
    """More tokens than the search keeps in LDS; all weights equal: the earliest stay."""
    r = np.random.default_rng(12)
    Hkv, D, B, n, keep = 2, 128, 128, 40001, 5000
    c, table, acc, tmax = evict_case(r, INT8, Hkv, D, B, [n], spare=40)
    to = np.full(table.shape, -1, np.int32)
    to[0, :40] = table.size + np.arange(40)
    acc[:, 1] = 0.25
    d, got, l1 = run_evict(ops, c, table, acc, [n], keep, 3, 100, n, to=to)
    assert l1[0] == keep
    ks = d.ks.read(np.float32).reshape(c.ks.shape)
    for h in range(Hkv):
        a = acc[table[0], h].reshape(-1)[:n].astype(np.float64)
        a = np.where(a > 0, a, 0)
        a[:3], a[n - 100:] = np.inf, np.inf
        kept = np.sort(np.lexsort((np.arange(n), -a))[:keep])
        assert np.array_equal(got[to[0, :40], h].reshape(-1)[:keep], acc[table[0], h].reshape(-1)[:n][kept], equal_nan=True)
        if h == 1:
            assert np.array_equal(kept, np.concatenate([np.arange(keep - 100), np.arange(n - 100, n)]))
        for j in (0, 7, 39):
            rows = kept[j * B:(j + 1) * B]
            sc = c.ks[table[0, rows // B], h].astype(np.float64)
            assert ks[to[0, j], h] == sc.max()
            want = encode(INT8, values(INT8, c.k[table[0, rows // B], h, rows % B]) * (sc / sc.max())[:, None])
            assert same_codes(INT8, d.k.read(np.uint8).reshape(c.k.shape)[to[0, j], h, :len(rows)], want)


@pytest.mark.parametrize("n,keep,first,last", [(2048, 600, 3, 0), (2049, 2000, 0, 70), (5000, 77, 4, 60), (8192, 3000, 0, 1), (8193, 8192, 1, 1), (20000, 1500, 2, 100)])
def test_evict_at_the_searchs_sizes(ops, n, keep, first, last):
    """As many weights a thread as there are registers for, at both ends; many equal ones around the last kept place; entries that are no blocks; a
    second sequence that stays whole."""
    r = np.random.default_rng(n)
    Hkv, D, B, lens = 2, 128, 128, [n, 60]
    need = (keep + B - 1) // B
    c, table, acc, tmax = evict_case(r, E4M3, Hkv, D, B, lens, spare=2 * need)
    acc[:, 1] = np.round(acc[:, 1] * 2) / 2
    to = np.full(table.shape, -1, np.int32)
    to[:, :need] = table.size + r.permutation(2 * need).reshape(2, need)
    table[0, [1, tmax // 2]] = -1, 1 << 20
    before = Cache.__new__(Cache)
    before.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()}
    d, got, l1 = run_evict(ops, before, table, acc, lens, keep, first, last, n, to=to)
    want = acc.copy()
    new = c.evict(want, table, np.array(lens), keep, first, last, to=to)
    assert np.array_equal(l1, new) and np.array_equal(got, want, equal_nan=True)
    check_pools(c, d)


@pytest.mark.parametrize("inside", [True, False])
def test_evict_sequences_a_few_at_a_time(ops, tune, inside):
    """Where the scratch holds a few sequences' lists and blocks only."""
    r = np.random.default_rng(13)
    Hkv, D, B, keep = 8, 128, 16, 150
    lens = [400] * 12
    need = (keep + B - 1) // B
    c, table, acc, tmax = evict_case(r, INT8, Hkv, D, B, lens, spare=12 * need)
    to = None
    if not inside:
        to = np.full(table.shape, -1, np.int32)
        to[:, :need] = table.size + np.arange(12 * need).reshape(12, need)
    tune(TUNE_SCRATCH_MIB, 1)
    before = Cache.__new__(Cache)
    before.__dict__ = {k: v.copy() if isinstance(v, np.ndarray) else v for k, v in c.__dict__.items()}
    d, got, l1 = run_evict(ops, before, table, acc, lens, keep, 1, 9, 400, to=to)
    want = acc.copy()
    new = c.evict(want, table, np.array(lens), keep, 1, 9, to=to)
    assert np.array_equal(l1, new) and np.array_equal(got, want, equal_nan=True)
    check_pools(c, d)
