"""The hybrid layers' calls (include/ns_layer.h) where rows, states or weights lie more than 2^32 bytes from their buffer's start."""
import numpy as np
import pytest

from layer_ref import F32, Layer, check_scan, elt_dtype, q4_weights, rms, scan, silu
from nextsycl_amd import DevBuf

pytestmark = pytest.mark.gpu
FAR = 1 << 23                      # floats between rows: 32 MiB


def spread(g, rows, stride):
    """Rows `stride` floats apart in a buffer of their own."""
    b = DevBuf(g, ((rows.shape[0] - 1) * stride + rows.shape[1]) * 4)
    for t, row in enumerate(rows):
        b.view(t * stride * 4, row.nbytes).write(row)
    return b


def gather(b, n, stride, width):
    return np.stack([b.read(np.float32, width, t * stride * 4) for t in range(n)])


@pytest.mark.parametrize("T,p0", [(140, 0), (140, 9)])
def test_prompt_rows_far_apart(ops, T, p0):
    g = ops.gpu
    H, P, N, G, K = 2, 32, 32, 1, 4
    L = Layer(H, P, N, G, K, seed=1)
    raw = np.random.default_rng(2).standard_normal((T, L.chan + H)).astype(np.float32)
    past = np.random.default_rng(3).standard_normal((3, L.chan)).astype(np.float32) * (p0 > 0)
    ring = np.full((4, L.chan), np.nan, np.float32)
    if p0:
        for k in range(3):
            ring[(p0 - 3 + k) % 4] = past[k]
    y, h, yb, hb = scan(L, raw[:, :L.chan], raw[:, L.chan:], past, np.zeros((H, P, N)))
    rows, w = spread(g, raw, FAR), [DevBuf.of(g, a) for a in (L.cw, L.cb, L.a, L.dtb, L.d)]
    yo, h1, sc = DevBuf(g, ((T - 1) * FAR + L.inner) * 4), DevBuf(g, H * P * N * 4), DevBuf(g, 4 * ops.ssm_prompt_scratch(T, H, P, N, G, K))
    ops.ssm_prompt(F32, rows, FAR, rows.view(L.chan * 4, rows.len - L.chan * 4), FAR, *w, DevBuf.of(g, ring), 4, p0, T, H, P, N, G, K, None, h1, yo, FAR, sc)
    g.sync()
    check_scan(gather(yo, T, FAR, L.inner), y, yb, F32, T, N, "y")
    check_scan(h1.read(np.float32).reshape(H, P, N), h[T], hb[T], F32, T, N, "state")


def test_step_states_and_rings_far_apart(ops):
    g = ops.gpu
    H, P, N, G, K, cap, nslots = 64, 64, 128, 1, 4, 40, 2100
    L = Layer(H, P, N, G, K, seed=4)
    slots = [2099, 5, 2050]
    raw = np.random.default_rng(5).standard_normal((3, L.chan + H)).astype(np.float32)
    state, rings = DevBuf(g, nslots * H * P * N * 4), DevBuf(g, nslots * cap * L.chan * 4)
    assert state.len > 1 << 32
    r = np.random.default_rng(6)
    h0, past = r.standard_normal((3, H, P, N)).astype(np.float32), r.standard_normal((3, 3, L.chan)).astype(np.float32)
    for i, s in enumerate(slots):
        state.view(s * h0[i].nbytes, h0[i].nbytes).write(h0[i])
        rings.view((s * cap + 17) * L.chan * 4, past[i].nbytes).write(past[i])
    w = [DevBuf.of(g, a) for a in (L.cw, L.cb, L.a, L.dtb, L.d)]
    rows, yo, row = DevBuf.of(g, raw), DevBuf(g, 3 * L.inner * 4), L.chan + H
    ops.ssm_step(F32, rows, row, rows.view(L.chan * 4, rows.len - L.chan * 4), row, *w, rings, cap, 20, 3, H, P, N, G, K, state, state, yo, L.inner, nslots=nslots,
                 slots=DevBuf.of(g, np.array(slots, np.int32)))
    g.sync()
    got = yo.read(np.float32).reshape(3, -1)
    for i, s in enumerate(slots):
        y, h, yb, hb = scan(L, raw[i:i + 1, :L.chan], raw[i:i + 1, L.chan:], past[i], h0[i])
        check_scan(got[i:i + 1], y, yb, F32, 1, N, "y")
        check_scan(state.read(np.float32, H * P * N, s * h0[i].nbytes).reshape(H, P, N), h[1], hb[1], F32, 1, N, "state")
        assert np.array_equal(rings.read(np.float32, L.chan, (s * cap + 20) * L.chan * 4), raw[i, :L.chan])


def test_norm_rows_far_apart(ops):
    """(float32 sums of 333 squares and an inverse root: 2^-18 of a value is far more than their roundings)"""
    g, D, T, far = ops.gpu, 333, 3, 600 << 20
    r = np.random.default_rng(7)
    y, z = r.standard_normal((T, D)).astype(np.float32), r.standard_normal((T, D)).astype(np.float32)
    yb, zb, ob = spread(g, y, far), spread(g, z, far), DevBuf(g, ((T - 1) * far + D) * 4)
    ops.norm_gated(F32, yb, far, zb, far, None, ob, far, T, D, 1, 1e-5)
    want = rms(y.astype(np.float64) * silu(z.astype(np.float64)), 1e-5)
    assert np.abs(gather(ob, T, far, D) - want).max() <= 2.0 ** -18 * np.abs(want).max()
    ops.norm_residual(F32, F32, yb, far, zb, far, zb, far, ob, far, T, D, 1e-5)
    s = y.astype(np.float64) + z
    assert np.abs(gather(zb, T, far, D) - s).max() <= 2.0 ** -24 * np.abs(s).max()
    assert np.abs(gather(ob, T, far, D) - rms(s, 1e-5)).max() <= 2.0 ** -18 * np.abs(rms(s, 1e-5)).max()


def test_q4_weights_past_32_bits(ops):
    """Weights of 0 but for a tile in front of 2^32 bytes and one behind."""
    g, K, group = ops.gpu, 4096, 32
    tile = 1024 + 32 * (128 // group)
    per = K // 128 * tile
    M = ((1 << 32) // per + 40) * 16
    w = DevBuf(g, ops.q4_bytes(M, K, group))
    w.fill(0x88)                               # nibbles of 8: weights of 0 whatever the scales (0x8888 is a small half)
    r = np.random.default_rng(8)
    x = r.standard_normal((2, K)).astype(np.float32)
    rows = {}
    for mt, kt in ((3, 7), (M // 16 - 2, 30)):
        t = np.concatenate([r.integers(0, 256, 1024, np.uint8), (r.uniform(0.01, 0.1, 16 * (128 // group))).astype(np.float16).view(np.uint8)])
        w.view(mt * per + kt * tile, tile).write(t)
        rows[mt] = (kt, q4_weights(t, 16, 128, group)[0])
    y = DevBuf(g, 2 * M * 4)
    ops.q4_product(F32, DevBuf.of(g, x), K, w, group, y, M, 2, M, K)
    got = y.read(np.float32).reshape(2, M)
    for mt, (kt, wt) in rows.items():
        part = x[:, kt * 128:kt * 128 + 128].astype(np.float64)
        # (128 products of 22 bits, summed in float32: 128 roundings of the sum of absolute values at most)
        assert (np.abs(got[:, mt * 16:mt * 16 + 16] - part @ wt.T) <= 2.0 ** -24 * 140 * (np.abs(part) @ np.abs(wt).T)).all()
        got[:, mt * 16:mt * 16 + 16] = 0.0
    assert not got.any()
