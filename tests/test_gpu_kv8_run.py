"""Caches of 8-bit values in blocks of tokens (include/ns_kv8.h) as a serving loop uses them: prompts, weights, eviction and tokens one
after another, recorded into graphs, from threads and two handles, on pools past 4 GiB, with many sequences over the same blocks."""
import ctypes as C
import threading

import numpy as np
import pytest

from kv8_ref import BF16, E4M3, F16, F32, INT8, Cache, from_type, to_type
from nextsycl_amd import DevBuf, Gpu
from nextsycl_amd.attn import Kv8, Ops
from test_gpu_kv8 import attend, back, check_pools, check_rows, filled, ints, on_gpu, prompt_close, rows_of, tables

pytestmark = pytest.mark.gpu
E = {F32: 4, F16: 2, BF16: 2}


def read_rows(qt, b, shape):
    return from_type(qt, b.read(np.float32 if qt == F32 else np.uint16)).reshape(shape)


# ---- all of them together

@pytest.mark.parametrize("form,qt,Hq,Hkv,D,B,inside", [(INT8, BF16, 8, 2, 128, 16, True), (E4M3, F16, 6, 2, 256, 32, True), (INT8, F32, 12, 4, 128, 64, False),
                                                       (E4M3, BF16, 4, 4, 256, 16, False)])
def test_a_serving_loop(ops, form, qt, Hq, Hkv, D, B, inside):
    """Two sequences' prompts stored, attended, their rows' weights summed; both shortened; then tokens, each stored and attended with its weights. The
    reference goes the same way, its eviction from the GPU's own sums (checked first: two sums a rounding apart may keep different tokens)."""
    r = np.random.default_rng(Hq + D + B)
    g, P, steps, keep = ops.gpu, [150, 61], 5, 40
    tmax = (max(P) + steps + B - 1) // B
    need = (keep + steps + B - 1) // B
    c = Cache(form, 2 * tmax + 2 * need, Hkv, B, D, seed=1)
    d, table = on_gpu(ops, c), tables(r, 2, tmax, 2 * tmax)
    T, start = sum(P), np.array([0, P[0], sum(P)], np.int32)
    k, ks, kv = rows_of(qt, r, T, Hkv, D, 0.7)
    v, vs, vv = rows_of(qt, r, T, Hkv, D, 0.7)
    q, qs, qv = rows_of(qt, r, T, Hq, D, 0.7, pad=8)
    kb, vb, qb, ob, acc = DevBuf.of(g, k), DevBuf.of(g, v), DevBuf.of(g, q), DevBuf(g, T * Hq * D * E[qt]), DevBuf(g, c.blocks * Hkv * B * 4)
    acc.fill(0xFF)
    tb, lens = ints(ops, table), ints(ops, [0, 0])
    ops.kv8_store(d, qt, kb, ks, vb, vs, T, tb, tmax, 2, max(P), lens, start=ints(ops, start))
    c.store(kv, vv, table, [0, 0], start, max(P))
    check_pools(c, d, "prompts")
    want = np.full((c.blocks, Hkv, B), np.nan)
    for s in range(2):
        a, n = int(start[s]), P[s]
        rows, seq = qb.view(a * qs * E[qt], qb.len - a * qs * E[qt]), tb.view(4 * s * tmax, 4 * tmax)
        ops.kv8_prompt(d, qt, rows, qs, n, seq, tmax, 0, Hq, ob.view(a * Hq * D * E[qt], n * Hq * D * E[qt]))
        ops.kv8_weights(d, qt, rows, qs, n, seq, tmax, 0, Hq, None, acc)
        ref, given = c.attend(qv[a:a + n], table, s, 0)
        c.give(None, want, table, s, 0, given)
        prompt_close(qt, read_rows(qt, ob, (T, Hq, D))[a:a + n], ref, qv[a:a + n], *c.tokens(table, s, n), D)

    def check_acc(tab, lens):
        got = acc.read(np.float32).reshape(want.shape)
        for s, n in enumerate(lens):
            for t in range(n):
                assert np.abs(got[tab[s, t // B], :, t % B] - want[tab[s, t // B], :, t % B]).max() <= 2.0 ** -16 * max(1.0, float(np.nanmax(want))), (s, t)
        return got

    got = check_acc(table, P)
    to = None
    if not inside:
        to = np.full(table.shape, -1, np.int32)
        to[:, :need] = 2 * tmax + r.permutation(2 * need).reshape(2, need)
    lens.write(np.array(P, np.int32))
    tob = None if to is None else ints(ops, to)
    ops.kv8_evict(d, acc, tb, tmax, 2, max(P), lens, lens, keep, first=2, last=8, to=tob)
    want = got.astype(np.float32)
    now = c.evict(want, table, np.array(P), keep, 2, 8, to=to, longest=max(P))
    assert np.array_equal(lens.read(np.int32), now) and np.array_equal(acc.read(np.float32).reshape(want.shape), want, equal_nan=True)
    check_pools(c, d, "eviction")
    table, tb = (table, tb) if inside else (to, tob)

    longest, want = keep + steps, want.astype(np.float64)
    out = DevBuf(g, 2 * Hq * D * E[qt])
    sc = DevBuf(g, max(4, 4 * ops.kv8_attend_scratch(2, 1, Hq, Hkv, D, longest, True)))
    for step in range(steps):
        k, ks, kv = rows_of(qt, r, 2, Hkv, D, 0.9)
        q, qs, qv = rows_of(qt, r, 2, Hq, D)
        kb, qb = DevBuf.of(g, k), DevBuf.of(g, q)
        ops.kv8_store(d, qt, kb, ks, kb, ks, 2, tb, tmax, 2, 1, lens)
        ops.kv8_attend(d, qt, qb, qs, 2, tb, tmax, 2, 1, longest, lens, Hq, out, sc, acc0=acc, acc1=acc)
        c.store(kv, kv, table, now, [0, 1, 2], 1)
        check_pools(c, d, "step %d" % step)
        rows = out.read(np.float32 if qt == F32 else np.uint16).reshape(2, Hq, D)
        for s in range(2):
            ref, given = c.attend(qv[s:s + 1], table, s, int(now[s]))
            c.give(want.copy(), want, table, s, int(now[s]), given)
            check_rows(qt, rows[s:s + 1], ref, qv[s:s + 1], *c.tokens(table, s, int(now[s]) + 1), D, what="step %d" % step)
        now = now + 1
        lens.write(now.astype(np.int32))
        check_acc(table, now)


# ---- graphs

def copies(ops, c, n):
    return [on_gpu(ops, c) for _ in range(n)]


def recorded(ops, call):
    h = C.c_void_p()
    ops.ok(ops.k.q35_graph_begin(ops.raw(), C.byref(h)), "graph begin")
    try:
        call()
    finally:
        ops.ok(ops.k.q35_graph_end(ops.raw(), h), "graph end")
    return h


@pytest.mark.parametrize("form,qt,Hq,Hkv,D,B,most", [(INT8, BF16, 16, 4, 128, 16, 1), (E4M3, F32, 12, 2, 256, 64, 3)])
def test_tokens_in_a_graph(form, qt, Hq, Hkv, D, B, most):
    """Recorded once for contexts up to 700, replayed as these grow past blocks, chunks and work-groups, eager calls on a second cache and waits between: the
    same bits each time."""
    gpu = Gpu.open(0)
    ops = Ops(gpu)
    try:
        r = np.random.default_rng(most)
        S, longest = 3, 700
        tmax = (longest + B - 1) // B
        table = tables(r, S, tmax, S * tmax)
        lens = np.array([30, 126, 400])
        c = filled(r, form, S * tmax, Hkv, B, D, table, lens)
        caches = copies(ops, c, 2)
        T = S * most
        tb, lb, st = ints(ops, table), ints(ops, lens), ints(ops, np.arange(S + 1) * most)
        kb, qb = DevBuf(gpu, T * Hkv * D * E[qt]), DevBuf(gpu, T * Hq * D * E[qt])
        sc = DevBuf(gpu, 4 * ops.kv8_attend_scratch(S, most, Hq, Hkv, D, longest, True))
        outs, accs = [DevBuf(gpu, T * Hq * D * E[qt]) for _ in range(2)], [DevBuf.of(gpu, np.zeros((c.blocks, Hkv, B), np.float32)) for _ in range(2)]

        def step(i):
            ops.kv8_store(caches[i], qt, kb, Hkv * D, kb, Hkv * D, T, tb, tmax, S, most, lb, start=st)
            ops.kv8_attend(caches[i], qt, qb, Hq * D, T, tb, tmax, S, most, longest, lb, Hq, outs[i], sc, start=st, acc0=accs[i], acc1=accs[i])

        h = recorded(ops, lambda: step(0))
        for rep, lens in enumerate(([30, 126, 400], [31, 128, 401], [47, 250, 512], [130, -1, 600], [700 - most, 0, 690])):
            lb.write(np.array(lens, np.int32))
            kb.write(to_type(qt, r.standard_normal((T, Hkv, D)) * 2.0 ** rep)[0])
            qb.write(to_type(qt, r.standard_normal((T, Hq, D)))[0])
            for o in outs:
                o.fill(0xFF)
            sc.fill(0xFF)
            gpu.sync()
            ops.ok(ops.k.q35_graph_launch(ops.raw(), h), "graph launch")
            gpu.sync()
            step(1)
            gpu.sync()
            bits = [[x.read(np.uint8) for x in (outs[i], accs[i], caches[i].k, caches[i].v, caches[i].ks, caches[i].vs)] for i in range(2)]
            assert all(np.array_equal(a, b) for a, b in zip(*bits)), rep
        ops.k.q35_graph_free(h)
    finally:
        gpu.close()


@pytest.mark.parametrize("inside", [True, False])
def test_a_prompt_its_weights_and_an_eviction_in_a_graph(inside):
    """Two graphs that use the library's scratch one after the other, replayed in turn with eager calls between."""
    gpu = Gpu.open(0)
    ops = Ops(gpu)
    try:
        r = np.random.default_rng(2)
        Hq, Hkv, D, B, T, p0, keep = 8, 4, 128, 32, 90, 300, 100
        n = p0 + T
        tmax, need = (n + B - 1) // B, (keep + B - 1) // B
        table = tables(r, 1, tmax, tmax)
        c = filled(r, INT8, tmax + need, Hkv, B, D, table, [n])
        to = np.full((1, tmax), -1, np.int32)
        to[0, :need] = tmax + np.arange(need)
        caches = copies(ops, c, 2)
        tb, tob, lb, l1 = ints(ops, table), ints(ops, to), ints(ops, [n]), [ints(ops, [0]) for _ in range(2)]
        qb, outs = DevBuf(gpu, T * Hq * D * 2), [DevBuf(gpu, T * Hq * D * 2) for _ in range(2)]
        accs = [DevBuf.of(gpu, np.zeros((c.blocks, Hkv, B), np.float32)) for _ in range(2)]
        pools = [x.copy() for x in (c.k, c.v, c.ks, c.vs)]

        def prompt(i):
            ops.kv8_prompt(caches[i], BF16, qb, Hq * D, T, tb, tmax, p0, Hq, outs[i])
            ops.kv8_weights(caches[i], BF16, qb, Hq * D, T, tb, tmax, p0, Hq, None, accs[i])

        def evict(i):
            ops.kv8_evict(caches[i], accs[i], tb, tmax, 1, n, lb, l1[i], keep, 2, 16, to=None if inside else tob)

        first, second = recorded(ops, lambda: prompt(0)), recorded(ops, lambda: evict(0))
        for rep in range(4):
            qb.write(to_type(BF16, r.standard_normal((T, Hq, D)) * (1 + rep))[0])
            for cache in caches:
                for b, x in zip((cache.k, cache.v, cache.ks, cache.vs), pools):
                    b.write(x)
            gpu.sync()
            ops.ok(ops.k.q35_graph_launch(ops.raw(), first), "graph launch")
            prompt(1)
            ops.ok(ops.k.q35_graph_launch(ops.raw(), second), "graph launch")
            gpu.sync()
            evict(1)
            gpu.sync()
            bits = [[x.read(np.uint8) for x in (outs[i], accs[i], l1[i], caches[i].k, caches[i].v, caches[i].ks, caches[i].vs)] for i in range(2)]
            assert all(np.array_equal(a, b) for a, b in zip(*bits)), rep
        ops.k.q35_graph_free(first)
        ops.k.q35_graph_free(second)
    finally:
        gpu.close()


# ---- sizes

@pytest.mark.parametrize("Hkv,G,D,B,S", [(8, 1, 128, 16, 90), (2, 4, 128, 16, 300), (4, 6, 256, 16, 70)])
def test_many_sequences_over_the_same_blocks(ops, Hkv, G, D, B, S):
    """More sequences than a work-group has threads; runs of more tokens than a wave holds table entries for (128 of 16 tokens)."""
    r = np.random.default_rng(S)
    n = 4600
    tmax = (n + B - 1) // B
    one = r.permutation(tmax).astype(np.int32)
    c = Cache(INT8, tmax, Hkv, B, D, seed=3)
    c.k[:], c.v[:] = (r.integers(-127, 128, c.k.shape).astype(np.int8).view(np.uint8) for _ in range(2))
    c.ks[:], c.vs[:] = (2.0 ** r.integers(-8, -5, c.ks.shape) for _ in range(2))
    lens = r.integers(0, n, S)
    lens[[0, 1, 2, S // 2, S - 1]] = [n - 1, 0, -1, 2048, n - 1]
    q, qs, qv = rows_of(F32, r, S, Hkv * G, D)
    raw = attend(ops, c, on_gpu(ops, c), F32, q, qs, np.tile(one, (S, 1)), lens, None, S, 1, Hkv * G, longest=n)
    k, v = c.tokens(one[None], 0, n)
    for s in range(S):
        if lens[s] < 0:
            assert np.isnan(raw[s]).all()                    # (0xFF bytes: as they were)
            continue
        m = int(lens[s]) + 1
        ref = np.empty((1, Hkv * G, D))
        for h in range(Hkv * G):
            x = k[:m, h // G] @ qv[s, h] * D ** -0.5
            w = np.exp(x - x.max())
            ref[0, h] = w @ v[:m, h // G] / w.sum()
        check_rows(F32, raw[s:s + 1], ref, qv[s:s + 1], k[:m], v[:m], D, what=str(s))


@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("n", [300, 1500, 9000])
@pytest.mark.parametrize("win", [0, 1000])
def test_entries_that_are_no_blocks_however_the_tokens_are_dealt(ops, qt, n, win):
    """A unit a work-group, a chunk a work-group, runs: keys and values of zeros for entries out of range and for those behind the table's end."""
    r = np.random.default_rng(n)
    H, D, B = 8, 128, 16
    tmax = (n + B - 1) // B
    table = r.permutation(tmax).astype(np.int32)[None]
    c = Cache(E4M3, tmax, H, B, D, seed=1)
    c.k[:], c.v[:] = (r.integers(0, 126, c.k.shape).astype(np.uint8) | (r.integers(0, 2, c.k.shape).astype(np.uint8) << 7) for _ in range(2))
    c.ks[:], c.vs[:] = (2.0 ** r.integers(-8, -5, c.ks.shape) for _ in range(2))
    bad = r.random(tmax) < 0.1
    c.k[table[0, bad]] = 0x7F                              # (nothing is read from them)
    c.v[table[0, bad]] = 0x7F
    table[0, bad] = r.choice([-1, tmax, 1 << 30, -(1 << 31)], bad.sum())
    c.k[table[0, -3:].clip(0, tmax - 1)] = 0x7F
    short = np.ascontiguousarray(table[:, :-3])
    q, qs, qv = rows_of(qt, r, 1, H, D)
    raw = attend(ops, c, on_gpu(ops, c), qt, q, qs, short, np.array([n - 1]), None, 1, 1, H, longest=n, win=win)
    ref, _ = c.attend(qv, short, 0, n - 1, win)
    check_rows(qt, raw, ref, qv, *c.tokens(short, 0, n), D)


def test_pools_past_4_gib(ops):
    """Blocks behind the first 4 GiB of each pool: every call as on a small pool, bit for bit."""
    r = np.random.default_rng(5)
    g, form, qt, Hq, Hkv, D, B = ops.gpu, E4M3, BF16, 16, 8, 256, 128
    tmax, blocks, T = 4, 16384 + 32, 300
    far = Kv8(form, blocks, Hkv, B, D, *(DevBuf(g, n) for n in [blocks * Hkv * B * D] * 2 + [blocks * Hkv * 4] * 2))
    near = Kv8(form, 32, Hkv, B, D, *(DevBuf(g, n) for n in [32 * Hkv * B * D] * 2 + [32 * Hkv * 4] * 2))
    table, to = np.array([[3, 17, 8, 30]]), np.array([[1, 5, 9, 20]])
    k, ks, _ = rows_of(qt, r, T, Hkv, D)
    q, qs, _ = rows_of(qt, r, T, Hq, D)
    kb, qb = DevBuf.of(g, k), DevBuf.of(g, q)
    got = []
    for cache, off in ((far, blocks - 32), (near, 0)):
        tb, tob, lb, zero = ints(ops, table + off), ints(ops, to + off), ints(ops, [T]), ints(ops, [0])
        acc = DevBuf(g, cache.blocks * Hkv * B * 4)
        ops.kv8_store(cache, qt, kb, ks, kb, ks, T, tb, tmax, 1, T, zero, start=ints(ops, [0, T]))
        out, one = DevBuf(g, T * Hq * D * 2), DevBuf(g, Hq * D * 2)
        ops.kv8_prompt(cache, qt, qb, qs, T, tb, tmax, 0, Hq, out)
        ops.kv8_weights(cache, qt, qb, qs, T, tb, tmax, 0, Hq, None, acc)
        ops.kv8_evict(cache, acc, tb, tmax, 1, T, lb, lb, 140, 2, 10, to=tob)
        ops.kv8_store(cache, qt, kb, ks, kb, ks, 1, tob, tmax, 1, 1, lb)
        sc = DevBuf(g, 4 * ops.kv8_attend_scratch(1, 1, Hq, Hkv, D, T, True))
        ops.kv8_attend(cache, qt, qb, qs, 1, tob, tmax, 1, 1, T, lb, Hq, one, sc, acc0=acc, acc1=acc)
        g.sync()
        rows, per = (to + off)[0, :2], Hkv * B
        bits = [out.read(np.uint8), one.read(np.uint8), lb.read(np.int32)]
        # (tokens 0 .. 140 of the two blocks that the eviction kept)
        for b, n in zip(rows, (B, 13)):
            bits += [x.read(np.uint8, per * D, int(b) * per * D).reshape(Hkv, B, D)[:, :n] for x in (cache.k, cache.v)]
            bits += [x.read(np.float32, Hkv, int(b) * Hkv * 4) for x in (cache.ks, cache.vs)]
            bits += [acc.read(np.float32, per, int(b) * per * 4).reshape(Hkv, B)[:, :n]]
        got.append(bits)
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    assert np.isfinite(from_type(qt, got[0][1].view(np.uint16))).all() and got[0][2][0] == 140


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("shift,pad", [(1, 1), (3, 7), (0, 3)])
def test_rows_at_any_element(ops, qt, shift, pad):
    """Rows that begin at no multiple of 16 bytes: the bits of aligned ones, from the token's attention and the weights."""
    r = np.random.default_rng(shift)
    g, Hq, Hkv, D, B, n, T = ops.gpu, 10, 2, 128, 16, 260, 9
    table = tables(r, 1, 17, 17)
    c = filled(r, E4M3, 17, Hkv, B, D, table, [n])
    d, tb = on_gpu(ops, c), ints(ops, table)
    q, qs, _ = rows_of(qt, r, T, Hq, D, pad=pad, shift=shift)
    flat = np.stack([q[shift + t * qs:][:Hq * D] for t in range(T)]).ravel()
    got = []
    for rows, at, stride in ((q, shift, qs), (flat, 0, Hq * D)):
        b = DevBuf.of(g, rows)
        v = b.view(at * E[qt], b.len - at * E[qt])
        out, accs = DevBuf(g, T * Hq * D * E[qt]), [DevBuf.of(g, np.zeros((17, Hkv, B), np.float32)) for _ in range(2)]
        sc = DevBuf(g, 4 * ops.kv8_attend_scratch(1, T, Hq, Hkv, D, n, True))
        ops.kv8_attend(d, qt, v, stride, T, tb, 17, 1, T, n, ints(ops, [n - T]), Hq, out, sc, start=ints(ops, [0, T]), acc1=accs[0])
        ops.kv8_weights(d, qt, v, stride, T, tb, 17, n - T, Hq, None, accs[1])
        got.append([x.read(np.uint8) for x in [out] + accs])
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_a_window_longer_than_any_sequence(ops):
    r = np.random.default_rng(3)
    g, Hq, Hkv, D, B, n, T = ops.gpu, 8, 2, 128, 32, 300, 6
    table = tables(r, 1, 10, 10)
    c = filled(r, INT8, 10, Hkv, B, D, table, [n])
    d, tb = on_gpu(ops, c), ints(ops, table)
    q, qs, _ = rows_of(F16, r, T, Hq, D)
    qb, got = DevBuf.of(g, q), []
    for win in (0, -5, n, (1 << 63) - 1):
        acc = DevBuf.of(g, np.zeros((10, Hkv, B), np.float32))
        raw = attend(ops, c, d, F16, q, qs, table, np.array([n - T]), np.array([0, T]), T, T, Hq, win=win, acc1=acc)
        out = DevBuf(g, T * Hq * D * 2)
        ops.kv8_prompt(d, F16, qb, qs, T, tb, 10, n - T, Hq, out, win=win)
        ops.kv8_weights(d, F16, qb, qs, T, tb, 10, n - T, Hq, acc, acc, win=win)
        got.append([raw, out.read(np.uint8), acc.read(np.uint8)])
    for other in got[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(got[0], other))


# ---- the same bits, whoever calls

class Loop:
    """CALLS rounds of prompt, weights and eviction into fresh blocks, each into outputs of its own."""
    CALLS = 60

    def __init__(self, ops, seed):
        r = np.random.default_rng(seed)
        g = ops.gpu
        self.ops, self.Hq, self.D, self.T, self.p0, self.keep = ops, 8, 128, 40 + 30 * seed, 500, 128
        n = self.p0 + self.T
        self.n, self.tmax = n, (n + 15) // 16
        table = tables(r, 1, self.tmax, self.tmax)
        c = filled(r, INT8, self.tmax + 8, 4, 16, 128, table, [n], seed=seed)
        to = np.full((1, self.tmax), -1, np.int32)
        to[0, :8] = self.tmax + np.arange(8)
        self.cache, self.table, self.to, self.lens, self.l1 = on_gpu(ops, c), ints(ops, table), ints(ops, to), ints(ops, [n]), ints(ops, [0])
        self.q = DevBuf.of(g, to_type(BF16, r.standard_normal((self.T, self.Hq, self.D)))[0])
        self.one, self.per = self.T * self.Hq * self.D * 2, c.blocks * 4 * 16 * 4
        self.y, self.acc = DevBuf(g, self.CALLS * self.one), DevBuf(g, self.CALLS * self.per)

    def call(self, i):
        o, acc = self.ops, self.acc.view(i * self.per, self.per)
        o.kv8_prompt(self.cache, BF16, self.q, self.Hq * self.D, self.T, self.table, self.tmax, self.p0, self.Hq, self.y.view(i * self.one, self.one))
        o.kv8_weights(self.cache, BF16, self.q, self.Hq * self.D, self.T, self.table, self.tmax, self.p0, self.Hq, None, acc)
        o.kv8_evict(self.cache, acc, self.table, self.tmax, 1, self.n, self.lens, self.l1, self.keep, 1, 30, to=self.to)

    def bits(self, i):
        return [self.y.read(np.uint8, self.one, i * self.one), self.acc.read(np.uint8, self.per, i * self.per)] + \
            [x.read(np.uint8) for x in (self.cache.k, self.cache.v, self.cache.ks, self.cache.vs)]


@pytest.mark.parametrize("handles", [1, 2])
def test_two_threads(ops, handles):
    """On one handle (calls in any order, one scratch) and on two (side by side): every round the bits of the first alone."""
    other = Gpu.open(0) if handles == 2 else None
    try:
        loops = [Loop(ops, 1), Loop(Ops(other) if other else ops, 2)]
        want = []
        for x in loops:
            x.acc.fill(0)
            x.call(0)
            x.ops.gpu.sync()
            want.append(x.bits(0))
        start, errors = threading.Barrier(2), []

        def run(x):
            try:
                start.wait(60)
                for i in range(x.CALLS):
                    x.call(i)
            except Exception as e:  # noqa: BLE001
                errors.append(e)

        threads = [threading.Thread(target=run, args=(x,)) for x in loops]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors
        for x, w in zip(loops, want):
            x.ops.gpu.sync()
            for i in range(x.CALLS):
                assert all(np.array_equal(a, b) for a, b in zip(x.bits(i), w)), i
        del loops, x
    finally:
        if other:
            other.close()


@pytest.mark.parametrize("qt,Hq,Hkv,D,most", [(BF16, 32, 8, 128, 1), (F32, 24, 4, 256, 4)])
def test_attention_gives_the_same_bits_every_time(ops, qt, Hq, Hkv, D, most):
    r = np.random.default_rng(D)
    S, B, lens = 5, 32, np.array([2000, 17, 900, 1500, 300])
    tmax = 64
    table = tables(r, S, tmax, S * tmax)
    c = filled(r, INT8, S * tmax, Hkv, B, D, table, lens + most)
    d = on_gpu(ops, c)
    q, qs, _ = rows_of(qt, r, S * most, Hq, D)
    first = None
    for _ in range(10):
        acc = DevBuf.of(ops.gpu, np.zeros((c.blocks, Hkv, B), np.float32))
        raw = attend(ops, c, d, qt, q, qs, table, lens, np.arange(S + 1) * most, S * most, most, Hq, acc1=acc)
        now = [raw, acc.read(np.uint8)]
        first = first or now
        assert all(np.array_equal(a, b) for a, b in zip(first, now))
