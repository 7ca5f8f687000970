"""Caches of 8-bit values in blocks of tokens (include/ns_kv8.h) at their edges: blocks that were never stored into, whose scales and codes hold anything at
all, not finite numbers among it; the bits that rows and weights keep, and rows of every magnitude; sequences longer than said; the largest sizes."""
import numpy as np
import pytest

from kv8_ref import BF16, E4M3, F16, F32, INT8, Cache, from_type, to_type, tolerance
from nextsycl_amd import DevBuf
from nextsycl_amd.attn import TUNE_PREFILL_SPLITS, TUNE_PREFILL_WAVES, Kv8
from test_gpu_kv8 import attend, check_pools, check_rows, filled, ints, on_gpu, prompt_close, rows_of, store, tables

pytestmark = pytest.mark.gpu
ANYTHING = [np.nan, np.inf, -np.inf, 1e30, 70000.0]


def unwritten(r, form, Hkv, B, D, table, n, what):
    """A cache of which only the table's own blocks are stored into; block 0 and the last are not, and no entry is them. The scales there: `what`."""
    blocks = table.max() + 2
    assert table.min() < 0 and not (table == 0).any()
    c = filled(r, form, blocks, Hkv, B, D, table, [n], sigma=0.7)
    for b in set(range(blocks)) - set(table.ravel()):
        c.ks[b], c.vs[b] = what, what
    return c


def holes(r, tmax, at):
    table = (1 + r.permutation(tmax)).astype(np.int32)[None]
    for e, x in at:
        table[0, e] = x
    return table


@pytest.mark.parametrize("what", ANYTHING)
@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt,Hq,Hkv,D,B,T,p0,win", [(BF16, 8, 2, 128, 16, 40, 100, 0), (F16, 4, 2, 256, 32, 150, 33, 0), (F32, 6, 3, 128, 64, 70, 300, 150),
                                                    (BF16, 4, 4, 128, 128, 12, 300, 0)])
def test_prompt_entries_that_are_no_blocks(ops, what, form, qt, Hq, Hkv, D, B, T, p0, win):
    """Keys and values of zeros, whatever block 0 holds."""
    r = np.random.default_rng(B)
    n = p0 + T
    tmax = (n + B - 1) // B
    table = holes(r, tmax, [(1, -1), (tmax - 1, 1 << 30)])
    c = unwritten(r, form, Hkv, B, D, np.where(table > tmax, -1, table), n, what)
    q, qs, qv = rows_of(qt, r, T, Hq, D, pad=8)
    ob = DevBuf(ops.gpu, T * Hq * D * (4 if qt == F32 else 2))
    ops.kv8_prompt(on_gpu(ops, c), qt, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, ob, win=win)
    ops.gpu.sync()
    ref, _ = c.attend(qv, table, 0, p0, win)
    prompt_close(qt, from_type(qt, ob.read(np.float32 if qt == F32 else np.uint16)).reshape(ref.shape), ref, qv, *c.tokens(table, 0, n), D)


@pytest.mark.parametrize("what", ANYTHING)
@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt,Hq,Hkv,D,B,T,p0,win", [(BF16, 32, 2, 128, 16, 40, 100, 0), (F16, 12, 2, 256, 32, 90, 33, 0), (F32, 24, 3, 128, 64, 70, 300, 150),
                                                    (BF16, 4, 4, 128, 128, 3, 300, 0)])
def test_weights_entries_that_are_no_blocks(ops, what, form, qt, Hq, Hkv, D, B, T, p0, win):
    """Their share of a row's sum is a key of zeros', whatever block 0 holds; nothing is written for them. (Many rows; few rows, as a token's.)"""
    r = np.random.default_rng(B + 1)
    n = p0 + T
    tmax = (n + B - 1) // B
    table = holes(r, tmax, [(1, -1), (tmax - 1, 1 << 30)])
    c = unwritten(r, form, Hkv, B, D, np.where(table > tmax, -1, table), n, what)
    q, qs, qv = rows_of(qt, r, T, Hq, D, pad=3)
    acc0 = r.uniform(0, 3, (c.blocks, Hkv, B)).astype(np.float32)
    want = np.full(acc0.shape, -1.0)
    c.give(acc0.astype(np.float64), want, table, 0, p0, c.attend(qv, table, 0, p0, win)[1])
    a1 = DevBuf.of(ops.gpu, np.full_like(acc0, -1))
    ops.kv8_weights(on_gpu(ops, c), qt, DevBuf.of(ops.gpu, q), qs, T, ints(ops, table), tmax, p0, Hq, DevBuf.of(ops.gpu, acc0), a1, win=win)
    ops.gpu.sync()
    got = a1.read(np.float32).reshape(acc0.shape)
    assert np.abs(got - want).max() <= 2.0 ** -17 * max(1.0, want.max())


# ---- what is lost on the way

@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,B,lens,counts,most,win", [(32, 8, 128, 32, [4000], [1], 1, 0), (8, 2, 128, 64, [300, 1999, 40], [1, 1, 1], 1, 0), (24, 4, 256, 16, [700, 90], [4, 2], 4, 0),
                                                             (64, 2, 128, 16, [1500], [2], 2, 800)])
def test_a_tokens_16_bit_rows_are_rounded_once(ops, form, qt, Hq, Hkv, D, B, lens, counts, most, win):
    """A row of two bytes a value is the sum x, within d of the exact one, rounded: no further from the exact one than that rounded is, and twice d. d as
    float32 rows': 2^-17 in the mean (weights of 22 bits, `tolerance`). With weights of 11 bits half rows lie 1.4 times as far off."""
    r = np.random.default_rng(Hq + B)
    ends = [a + b for a, b in zip(lens, counts)]
    S, tmax = len(lens), max((e + B - 1) // B for e in ends)
    table = tables(r, S, tmax, S * tmax)
    c = filled(r, form, S * tmax, Hkv, B, D, table, ends)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q, qs, qv = rows_of(qt, r, int(start[-1]), Hq, D)
    raw = attend(ops, c, on_gpu(ops, c), qt, q, qs, table, lens, start, int(start[-1]), most, Hq, win=win)
    ref = np.concatenate([c.attend(qv[start[s]:start[s + 1]], table, s, lens[s], win)[0] for s in range(S)])
    rounded = to_type(qt, ref)[1]
    assert np.linalg.norm(from_type(qt, raw) - ref) <= np.linalg.norm(rounded - ref) + 2 * 2.0 ** -17 * np.linalg.norm(ref)


def one_prompt(r, form, qt, Hq, Hkv, D, B, T, p0, rows=1.0, keys=0.7):
    n = p0 + T
    tmax = (n + B - 1) // B
    table = tables(r, 1, tmax, tmax)
    c = Cache(form, tmax, Hkv, B, D, seed=B)
    k, v = (r.standard_normal((n, Hkv, D)) * sigma * np.exp(0.4 * r.standard_normal((1, Hkv, D))) for sigma in (keys, 1.0))
    c.store(k, v, table, [0], [0, n], n)
    q, qs, _ = rows_of(F32, r, T, Hq, D)
    q, qv = to_type(qt, q.reshape(T, Hq, D) * np.float32(rows))
    return c, table, q, qv


def run_prompt(ops, c, qt, q, table, p0, Hq, win=0, scale=0.0):
    ob = DevBuf(ops.gpu, q.shape[0] * Hq * c.D * (4 if qt == F32 else 2))
    ops.kv8_prompt(on_gpu(ops, c), qt, DevBuf.of(ops.gpu, q), Hq * c.D, q.shape[0], ints(ops, table), table.shape[1], p0, Hq, ob, win=win, scale=scale)
    ops.gpu.sync()
    return ob.read(np.float32 if qt == F32 else np.uint16).reshape(q.shape)


def check_prompt(qt, raw, ref, qv, k, v, D, scale=0.0, what=""):
    """A prompt's rows as a token's (`tolerance`), but for what sums up beside 16-bit rows: numerator and sum of a row carry the same weights of 11 bits there, and
    sum w (1 + d) v / sum w (1 + d) moves by sum w d (v - mean) / sum w, twice vmax 2^-11 at most."""
    got = from_type(qt, raw)
    Hq, Hkv = qv.shape[1], k.shape[1]
    reach = max(float((np.abs(qv[:, h]) @ np.abs(k[:, h * Hkv // Hq]).T).max()) for h in range(Hq)) * (scale or D ** -0.5) * np.log2(np.e)
    vmax = float(np.abs(v).max())
    tol, rel = tolerance(qt, ref, reach, vmax, D, len(k))
    tol += 0.0 if qt == F32 else vmax * 2.0 ** -11
    assert np.isfinite(got).all(), what
    assert np.abs(got - ref).max() <= tol, "%s: %.3g (<= %.3g)" % (what, np.abs(got - ref).max(), tol)
    assert np.linalg.norm(got - ref) <= rel * np.linalg.norm(ref), "%s: relative L2 %.3g (<= %.3g)" % (what, np.linalg.norm(got - ref) / np.linalg.norm(ref), rel)


LONG = [  # Hq, Hkv, D, B, T, p0, window, waves, splits
    (8, 2, 128, 64, 17, 300, 0, 0, 0),
    (6, 3, 256, 16, 33, 70, 0, 0, 0),
    (16, 2, 128, 32, 40, 2000, 0, 0, 0),
    (8, 2, 256, 64, 40, 2000, 0, 0, 0),
    (8, 8, 128, 32, 300, 0, 0, 8, 0),
    (4, 4, 256, 128, 200, 31, 0, 8, 0),
    (10, 2, 128, 16, 150, 500, 100, 4, 3),
    (12, 2, 256, 32, 70, 900, 0, 4, 2),
    (12, 3, 128, 32, 90, 700, 0, 16, 2),
    (12, 3, 128, 32, 200, 100, 64, 12, 0),
    (8, 1, 256, 32, 60, 300, 0, 16, 0),
]


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,B,T,p0,win,waves,splits", LONG)
def test_prompts_of_more_than_16_rows_keep_a_tokens_bits(ops, tune, form, qt, Hq, Hkv, D, B, T, p0, win, waves, splits):
    """Float32 rows 22 bits of themselves and of their weights, whatever form the pass takes; 16-bit rows all of theirs."""
    r = np.random.default_rng(T + D)
    c, table, q, qv = one_prompt(r, form, qt, Hq, Hkv, D, B, T, p0)
    if waves:
        tune(TUNE_PREFILL_WAVES, waves)
    if splits:
        tune(TUNE_PREFILL_SPLITS, splits)
    raw = run_prompt(ops, c, qt, q, table, p0, Hq, win)
    check_prompt(qt, raw, c.attend(qv, table, 0, p0, win)[0], qv, *c.tokens(table, 0, p0 + T), D)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("qt,rows,keys", [(F32, 2.0 ** 18, 2.0 ** -18), (BF16, 2.0 ** 18, 2.0 ** -18), (F16, 2.0 ** 11, 2.0 ** -11), (F32, 2.0 ** -14, 2.0 ** 13), (BF16, 2.0 ** -14, 2.0 ** 13),
                                          (F16, 2.0 ** -12, 2.0 ** 12)])
@pytest.mark.parametrize("Hq,Hkv,D,B,T,p0", [(8, 2, 128, 32, 40, 300), (4, 2, 256, 64, 40, 60), (16, 2, 128, 16, 20, 3000), (8, 1, 256, 16, 30, 2000)])
def test_prompts_rows_of_any_range(ops, form, qt, rows, keys, Hq, Hkv, D, B, T, p0):
    """Rows far outside a half's range, or where its steps are wide, against keys that bring the scores back."""
    r = np.random.default_rng(T)
    c, table, q, qv = one_prompt(r, form, qt, Hq, Hkv, D, B, T, p0, rows, keys)
    check_prompt(qt, run_prompt(ops, c, qt, q, table, p0, Hq), c.attend(qv, table, 0, p0)[0], qv, *c.tokens(table, 0, p0 + T), D)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("rows,scale", [(2.0 ** 122, 2.0 ** -125), (2.0 ** 100, 2.0 ** -103), (2.0 ** -100, 2.0 ** 97)])
def test_prompts_at_the_ends_of_float32(ops, form, rows, scale):
    """Rows of every magnitude, a scale that brings the scores back (below 2^-107 the rows keep fewer bits: not asked for here); rows of zeros; NaN and
    infinities stay in their row and head."""
    Hq, Hkv, D, B, T, p0 = 4, 2, 128, 16, 24, 60
    r = np.random.default_rng(5)
    c, table, q, _ = one_prompt(r, form, F32, Hq, Hkv, D, B, T, p0, 1.0, 0.7)
    q = q * np.float32(rows)
    q[3] = 0
    qv = q.astype(np.float64)
    ref, _ = c.attend(qv, table, 0, p0, scale=scale)
    k, v = c.tokens(table, 0, p0 + T)
    check_prompt(F32, run_prompt(ops, c, F32, q, table, p0, Hq, scale=scale), ref, qv, k, v, D, scale)
    q[5, 1, 7], q[9, 2, 3], q[11, 0, 2] = np.nan, np.inf, -np.inf
    raw = run_prompt(ops, c, F32, q, table, p0, Hq, scale=scale)
    bad = np.zeros((T, Hq), bool)
    bad[[5, 9, 11], [1, 2, 0]] = True
    assert np.isnan(raw[bad]).all()
    rel = np.linalg.norm(raw[~bad].astype(np.float64) - ref[~bad]) / np.linalg.norm(ref[~bad])
    assert rel <= 2.0 ** -17 + 2.0 ** -24


# ---- sequences longer than said

@pytest.mark.parametrize("Hq,Hkv,S,most,longest,lens", [(8, 4, 4, 2, 60, [40, -5, 100, 700]), (64, 2, 2, 3, 100, [3000, 90]), (4, 1, 1, 1, 900, [5000]), (16, 8, 40, 1, 9000, [300, 12000, 9001] + 37 * [50]),
                                                        (32, 1, 1, 16, 500, [2000])])
@pytest.mark.parametrize("acc0", [True, False])
def test_weights_of_tokens_past_longest(ops, Hq, Hkv, S, most, longest, lens, acc0):
    """acc1 = acc0 + what is given for every token in front of a sequence's end, those from `longest` on too - nothing is given to them -, whether a work-group sums
    up its own unit, the chunks are a work-group's each or lie end to end."""
    r = np.random.default_rng(longest)
    D, B = 128, 16
    n = max(lens) + most
    tmax = (n + B - 1) // B - 1                          # (and the last tokens lie behind the table)
    one = tables(r, 1, tmax, tmax)[0]
    c = Cache(INT8, S * tmax, Hkv, B, D, seed=2)
    c.k[:], c.v[:] = (r.integers(-127, 128, c.k.shape).astype(np.int8).view(np.uint8) for _ in range(2))
    c.ks[:], c.vs[:] = (2.0 ** r.integers(-8, -5, c.ks.shape) for _ in range(2))
    table = (one + np.arange(S)[:, None] * tmax).astype(np.int32)
    start = np.arange(S + 1) * most
    q, qs, qv = rows_of(F32, r, S * most, Hq, D)
    was = r.uniform(0, 3, (c.blocks, Hkv, B)).astype(np.float32)
    want = np.full(was.shape, -1.0)
    a1 = DevBuf.of(ops.gpu, np.full_like(was, -1))
    attend(ops, c, on_gpu(ops, c), F32, q, qs, table, lens, start, S * most, most, Hq, longest=longest, acc0=DevBuf.of(ops.gpu, was) if acc0 else None, acc1=a1)
    for s in range(S):
        if lens[s] >= 0:
            _, given = c.attend(qv[start[s]:start[s + 1]], table, s, lens[s], longest=longest)
            c.give(was.astype(np.float64) if acc0 else None, want, table, s, lens[s], given)
    assert np.abs(a1.read(np.float32).reshape(was.shape) - want).max() <= 2.0 ** -17 * max(1.0, want.max())


# ---- rows of every magnitude that float32 has

ENDS = [(2.0 ** 123, 2.0 ** -126), (2.0 ** 100, 2.0 ** -103), (2.0 ** -104, 2.0 ** 101)]


def end_rows(r, form, Hq, Hkv, D, B, T, p0, rows):
    """The largest value 2^127 and more where rows are 2^123; a row of zeros."""
    c, table, q, _ = one_prompt(r, form, F32, Hq, Hkv, D, B, T, p0)
    q = np.clip(q, -15.5, 15.5) * np.float32(rows)
    q[0, 0, 3] = np.float32(15.5) * np.float32(rows)
    if T > 2:
        q[2] = 0
    return c, table, q, q.astype(np.float64)


@pytest.mark.parametrize("form", [INT8, E4M3])
@pytest.mark.parametrize("rows,scale", ENDS)
@pytest.mark.parametrize("Hq,Hkv,D,B,T,p0", [(8, 2, 128, 32, 1, 500), (4, 2, 256, 16, 9, 60), (6, 2, 128, 64, 40, 300), (4, 1, 256, 32, 20, 100)])
def test_rows_at_the_ends_of_float32(ops, form, rows, scale, Hq, Hkv, D, B, T, p0):
    """A scale, or keys, that bring the scores back: tokens' rows (up to 16), prompts, weights."""
    r = np.random.default_rng(T)
    c, table, q, qv = end_rows(r, form, Hq, Hkv, D, B, T, p0, rows)
    ref, given = c.attend(qv, table, 0, p0, scale=scale)
    k, v = c.tokens(table, 0, p0 + T)
    check_prompt(F32, run_prompt(ops, c, F32, q, table, p0, Hq, scale=scale), ref, qv, k, v, D, scale, "prompt")
    want = np.zeros((c.blocks, Hkv, B))
    c.give(None, want, table, 0, p0, given)
    acc = DevBuf.of(ops.gpu, np.zeros(want.shape, np.float32))
    if T <= 16:
        raw = attend(ops, c, on_gpu(ops, c), F32, q, Hq * D, table, np.array([p0]), np.array([0, T]), T, T, Hq, scale=scale, acc1=acc)
        check_prompt(F32, raw, ref, qv, k, v, D, scale, "tokens")
        assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * max(1.0, want.max())
    ops.kv8_weights(on_gpu(ops, c), F32, DevBuf.of(ops.gpu, q), Hq * D, T, ints(ops, table), table.shape[1], p0, Hq, None, acc, scale=scale)
    assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * max(1.0, want.max())


@pytest.mark.parametrize("T", [1, 40])
def test_rows_that_a_small_scale_makes_nothing_of(ops, T):
    """Scores of 2^-140 and less: a mean of all that a row sees, also where tokens are masked."""
    r = np.random.default_rng(T)
    c, table, q, qv = end_rows(r, INT8, 4, 2, 128, 16, T, 90, 2.0 ** -110)
    scale = 2.0 ** -60
    ref, given = c.attend(qv, table, 0, 90, 50, scale=scale)
    k, v = c.tokens(table, 0, 90 + T)
    check_prompt(F32, run_prompt(ops, c, F32, q, table, 90, 4, 50, scale), ref, qv, k, v, 128, scale)
    want = np.zeros((c.blocks, 2, 16))
    c.give(None, want, table, 0, 90, given)
    acc = DevBuf.of(ops.gpu, np.zeros(want.shape, np.float32))
    ops.kv8_weights(on_gpu(ops, c), F32, DevBuf.of(ops.gpu, q), 512, T, ints(ops, table), table.shape[1], 90, 4, None, acc, win=50, scale=scale)
    assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * max(1.0, want.max())


@pytest.mark.parametrize("qt,Hq,Hkv,D,T,p0", [(BF16, 8, 2, 128, 40, 260), (F32, 8, 8, 128, 300, 3), (F16, 4, 2, 256, 150, 50)])
def test_a_prompts_window_longer_than_any_sequence(ops, qt, Hq, Hkv, D, T, p0):
    """The bits of none, up to the longest there is to say."""
    r = np.random.default_rng(T)
    c, table, q, _ = one_prompt(r, INT8, qt, Hq, Hkv, D, 32, T, p0)
    first = run_prompt(ops, c, qt, q, table, p0, Hq)
    for win in (-1, 1 << 31, (1 << 62) + 3, (1 << 63) - 1):
        assert np.array_equal(run_prompt(ops, c, qt, q, table, p0, Hq, win), first), win


# ---- the largest sizes

@pytest.mark.parametrize("G,D,n,T", [(4096, 128, 40, 1), (4096, 128, 150, 2), (3001, 128, 70, 17), (4096, 256, 33, 20), (1025, 256, 300, 5)])
def test_thousands_of_query_heads_a_key_head(ops, G, D, n, T):
    r = np.random.default_rng(G + T)
    c, table, q, qv = one_prompt(r, INT8, F16, G, 1, D, 16, T, n - T)
    ref, given = c.attend(qv, table, 0, n - T)
    k, v = c.tokens(table, 0, n)
    check_prompt(F16, run_prompt(ops, c, F16, q, table, n - T, G), ref, qv, k, v, D, what="prompt")
    want = np.zeros((c.blocks, 1, 16))
    c.give(None, want, table, 0, n - T, given)
    accs = [DevBuf.of(ops.gpu, np.zeros(want.shape, np.float32)) for _ in range(2)]
    if T <= 16:
        raw = attend(ops, c, on_gpu(ops, c), F16, q, G * D, table, np.array([n - T]), np.array([0, T]), T, T, G, acc1=accs[0])
        check_prompt(F16, raw, ref, qv, k, v, D, what="tokens")
        assert np.abs(accs[0].read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * want.max()
    ops.kv8_weights(on_gpu(ops, c), F16, DevBuf.of(ops.gpu, q), G * D, T, ints(ops, table), table.shape[1], n - T, G, None, accs[1])
    assert np.abs(accs[1].read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17 * want.max()


@pytest.mark.parametrize("longest", [30, 2100])
def test_65535_sequences(ops, longest):
    """Most of them without a row or a length; a unit a work-group, and runs."""
    r = np.random.default_rng(longest)
    S, Hq, Hkv, D, B = 65535, 2, 1, 128, 16
    tmax = (longest + B - 1) // B
    some = [0, 1, 63, 64, 1023, 1024, 40000, 65533, 65534]
    lens = np.full(S, -1)
    lens[some] = [longest - 1, 0, 7, longest - 1, 16, longest // 2, 3, 15, longest - 2]
    table = np.full((S, tmax), -1, np.int32)
    table[some] = np.arange(len(some) * tmax).reshape(len(some), tmax)
    start = np.zeros(S + 1, np.int64)
    start[1:] = np.cumsum(lens >= 0)
    c = Cache(INT8, len(some) * tmax, Hkv, B, D, seed=1)
    c.k[:], c.v[:] = (r.integers(-127, 128, c.k.shape).astype(np.int8).view(np.uint8) for _ in range(2))
    c.ks[:], c.vs[:] = (2.0 ** r.integers(-8, -5, c.ks.shape) for _ in range(2))
    d = on_gpu(ops, c)
    q, qs, qv = rows_of(F32, r, len(some), Hq, D)
    k, ks, kv = rows_of(F32, r, len(some), Hkv, D)
    store(ops, c, d, F32, k, ks, k, ks, len(some), table, lens, start, 1)
    one = [0 if i == 0 else i for i in range(len(some) + 1)]
    c.store(kv, kv, table[some], lens[some], one, 1)
    check_pools(c, d)
    acc = DevBuf.of(ops.gpu, np.zeros((c.blocks, Hkv, B), np.float32))
    raw = attend(ops, c, d, F32, q, qs, table, lens, start, len(some), 1, Hq, longest=longest, acc1=acc)
    want = np.zeros((c.blocks, Hkv, B))
    for i, s in enumerate(some):
        ref, given = c.attend(qv[i:i + 1], table, s, int(lens[s]))
        check_rows(F32, raw[i:i + 1], ref, qv[i:i + 1], *c.tokens(table, s, int(lens[s]) + 1), D, what=str(s))
        c.give(None, want, table, s, int(lens[s]), given)
    assert np.abs(acc.read(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -17
    # and all of them shortened, in groups as the scratch holds them
    l1 = ints(ops, np.full(S, 77))
    ops.kv8_evict(d, acc, ints(ops, table), tmax, S, longest, ints(ops, lens), l1, 12, 1, 3)
    sums = acc.read(np.float32).reshape(want.shape)
    assert np.array_equal(l1.read(np.int32), np.minimum(lens, 12)) and np.isfinite(sums).all()


def test_32767_key_heads(ops):
    r = np.random.default_rng(8)
    H, D, B, n = 32767, 128, 16, 21
    table = np.array([[1, 0]], np.int32)
    k = DevBuf.of(ops.gpu, to_type(BF16, r.standard_normal((n, H * D), np.float32))[0])
    cache = Kv8.new(ops.gpu, INT8, 2, H, B, D)
    ops.kv8_store(cache, BF16, k, H * D, k, H * D, n, ints(ops, table), 2, 1, n, ints(ops, [0]), start=ints(ops, [0, n]))
    out, acc = DevBuf(ops.gpu, H * D * 2), DevBuf(ops.gpu, 2 * H * B * 4)
    acc.fill(0)
    lens = ints(ops, [n - 1])
    sc = DevBuf(ops.gpu, max(4, 4 * ops.kv8_attend_scratch(1, 1, H, H, D, n, True)))
    q = k.view(H * D * 2 * (n - 1), H * D * 2)
    ops.kv8_attend(cache, BF16, q, H * D, 1, ints(ops, table), 2, 1, 1, n, lens, H, out, sc, acc1=acc)
    prompt, many = DevBuf(ops.gpu, n * H * D * 2), DevBuf(ops.gpu, 2 * H * B * 4)
    many.fill(0)
    ops.kv8_prompt(cache, BF16, k, H * D, n, ints(ops, table), 2, 0, H, prompt)
    ops.kv8_weights(cache, BF16, k, H * D, n, ints(ops, table), 2, 0, H, None, many)
    ops.gpu.sync()
    sums = acc.read(np.float32).reshape(2, H, B)
    whole = sums[1].astype(np.float64).sum(1) + sums[0, :, :n - B].astype(np.float64).sum(1)
    assert np.abs(whole - 1.0).max() <= 2.0 ** -17                      # (a row's weights)
    total = many.read(np.float32).reshape(2, H, B)
    total = total[1].astype(np.float64).sum(1) + total[0, :, :n - B].astype(np.float64).sum(1)
    assert np.abs(total - n).max() <= n * 2.0 ** -17
    # some heads against the definition; the prompt's last row is the token's, but for its weights' bits
    codes, scale = (cache.k.read(np.uint8).view(np.int8).reshape(2, H, B, D), cache.ks.read(np.float32).reshape(2, H))
    vals = from_type(BF16, k.read(np.uint16)).reshape(n, H, D)
    got, last = from_type(BF16, out.read(np.uint16)).reshape(H, D), from_type(BF16, prompt.read(np.uint16, H * D, (n - 1) * H * D * 2)).reshape(H, D)
    for h in (0, 1, 255, 16383, 16384, 32766):
        x = np.concatenate([codes[1, h] * float(scale[1, h]), codes[0, h, :n - B] * float(scale[0, h])])
        w = np.exp(x @ vals[n - 1, h] * D ** -0.5 - (x @ vals[n - 1, h] * D ** -0.5).max())
        ref = w @ x / w.sum()
        assert np.abs(got[h] - ref).max() <= (2.0 ** -8 + 2.0 ** -17) * np.abs(x).max() and np.abs(last[h] - ref).max() <= (2.0 ** -8 + 2.0 ** -10) * np.abs(x).max()
    # kept: 9 tokens a head
    ops.kv8_evict(cache, many, ints(ops, table), 2, 1, n, ints(ops, [n]), lens, 9, 1, 2)
    assert lens.read(np.int32)[0] == 9
