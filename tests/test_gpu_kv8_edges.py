"""Caches of 8-bit values in blocks of tokens (include/ns_kv8.h) where a call meets what nothing wrote: scales and codes of blocks that were never
stored into hold anything at all, not finite numbers among it."""
import numpy as np
import pytest

from kv8_ref import BF16, E4M3, F16, F32, INT8, from_type, to_type
from nextsycl_amd import DevBuf
from test_gpu_kv8 import attend, filled, ints, on_gpu, prompt_close, rows_of, tables

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
