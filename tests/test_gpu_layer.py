"""The norms around a block (ns_norm_gated, ns_norm_residual), the 4-bit products (ns_q4_pack, ns_q4_product) and a whole
layer of them, against float64."""
import ctypes as C

import numpy as np
import pytest

from layer_ref import BF16, F16, F32, ROUND, TINY, U32, Layer, elt_dtype, from_type, q4_weights, rms, scan, silu, to_type
from nextsycl_amd import DevBuf, Error, Gpu
from nextsycl_amd.attn import Ops

pytestmark = pytest.mark.gpu
E = {F32: 4, F16: 2, BF16: 2}
TYPES = [F32, F16, BF16]


def rows(qt, T, D, stride, seed, sigma=1.0):
    """(raw [T][stride] for the GPU, its first D columns as float64)."""
    raw, val = to_type(qt, np.random.default_rng(seed).standard_normal((T, stride)) * sigma)
    return raw, val[:, :D].astype(np.float64)


def near(got, ref, qt, roundings, what):
    """Every value within `roundings` float32 roundings and its own type's."""
    assert np.isfinite(got).all(), what
    err, tol = np.abs(got.astype(np.float64) - ref), (roundings * U32 + ROUND[qt]) * np.abs(ref) + TINY[qt] + 1e-30
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), "%s: %s is %.9g, should be %.9g" % (what, at, got[at], ref[at])


# a sum of squares: W additions in some tree of float32 (W / lanes + 6 of them in line), its mean, root and quotient; halved by the root
def norm_roundings(W):
    return 10 + min(W, 64 + W // 64)


# T, D, groups, pads of y, z, out; the last: longer than a work-group's registers hold
GATED = [(1, 64, 1, 0, 0, 0), (3, 8192, 8, 0, 0, 0), (5, 145, 1, 0, 0, 0), (2, 1000, 8, 8, 16, 24), (4, 4096, 1, 0, 8, 0), (2, 12, 4, 1, 2, 3), (1, 1, 1, 0, 0, 0),
         (70, 48, 3, 0, 0, 0), (2, 16384, 1, 0, 0, 0), (1, 33000, 1, 8, 8, 8), (2, 4099, 1, 5, 0, 1), (300, 256, 2, 0, 256, 0), (1, 9001, 1, 0, 0, 0)]


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("T,D,G,py,pz,po", GATED)
def test_norm_gated(ops, qt, order, T, D, G, py, pz, po):
    g, eps = ops.gpu, 1e-5
    y, yv = rows(qt, T, D, D + py, 1)
    z, zv = rows(qt, T, D, D + pz, 2, 2.0)
    w = (1.0 + 0.1 * np.random.default_rng(3).standard_normal(D)).astype(np.float32)
    gate = silu(zv)
    part = lambda v: rms(v.reshape(T, G, -1), eps).reshape(T, D)  # noqa: E731
    for weight in (w, None):
        ref = part(yv * (1.0 if order else gate)) * (1.0 if weight is None else weight) * (gate if order else 1.0)
        out = DevBuf(g, T * (D + po) * E[qt])
        out.fill(0xFF)
        wb = None if weight is None else DevBuf.of(g, weight)
        ops.norm_gated(qt, DevBuf.of(g, y), D + py, DevBuf.of(g, z), D + pz, wb, out, D + po, T, D, G, eps, order)
        got = out.read(elt_dtype(qt)).reshape(T, D + po)
        # (silu of an exponential and a quotient: 8 more, and 4 for an exponent of a few units)
        near(from_type(qt, np.ascontiguousarray(got[:, :D])), ref, qt, norm_roundings(D // G) + 12 + 2 * np.abs(zv).max(), "gated")
        rest = np.ascontiguousarray(got[:, D:])
        assert (rest.view(np.uint8) == 0xFF).all()
    # into y, and into z
    for into in (0, 1):
        yb, zb = DevBuf.of(g, y), DevBuf.of(g, z)
        dst, stride = (yb, D + py) if into == 0 else (zb, D + pz)
        ops.norm_gated(qt, yb, D + py, zb, D + pz, wb, dst, stride, T, D, G, eps, order)
        again = dst.read(elt_dtype(qt)).reshape(T, stride)[:, :D]
        assert np.array_equal(again.view(np.uint8 if qt else np.uint32), got[:, :D].view(np.uint8 if qt else np.uint32)) or np.array_equal(again, got[:, :D])


RESIDUAL = [(1, 4096, 0), (3, 5120, 0), (5, 145, 0), (2, 1000, 8), (1, 1, 0), (4, 33, 3), (2, 16384, 0), (1, 40000, 8), (300, 64, 0), (2, 9001, 0)]


@pytest.mark.parametrize("qt,rt", [(F32, F32), (F16, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("T,D,pad", RESIDUAL)
def test_norm_residual(ops, qt, rt, T, D, pad):
    g, eps, scale, s = ops.gpu, 1e-6, 0.22, D + pad
    r = np.random.default_rng(D)
    x, xv = rows(qt, T, D, s, 1)
    h, hv = rows(rt, T, D, s, 2, 3.0)
    vec = [(1.0 + 0.1 * r.standard_normal(D)).astype(np.float32) for _ in range(3)]
    xb, hb = DevBuf.of(g, x), DevBuf.of(g, h)
    for post, gate, pre in ((None, None, vec[2]), (vec[0], None, vec[2]), (None, vec[1], None), (vec[0], vec[1], vec[2])):
        v = rms(xv, eps) * post if post is not None else xv
        v = scale * (v * gate if gate is not None else v)
        ref = hv + v
        out = rms(ref, eps) * (1.0 if pre is None else pre)
        h1, o = DevBuf(g, T * s * E[rt]), DevBuf(g, T * s * E[qt])
        h1.fill(0xFF)
        o.fill(0xFF)
        opt = lambda a: None if a is None else DevBuf.of(g, a)  # noqa: E731
        ops.norm_residual(qt, rt, xb, s, hb, s, h1, s, o, s, T, D, eps, scale, post=opt(post), gate=opt(gate), pre=opt(pre))
        gs, go = h1.read(elt_dtype(rt)).reshape(T, s), o.read(elt_dtype(qt)).reshape(T, s)
        # a sum of two: its error is relative to both
        n = norm_roundings(D)
        err = np.abs(from_type(rt, np.ascontiguousarray(gs[:, :D])) - ref)
        slack = U32 * (n + 6) * (np.abs(v) + np.abs(hv)) + ROUND[rt] * np.abs(ref) + TINY[rt]
        assert (err <= slack).all()
        err = np.abs(from_type(qt, np.ascontiguousarray(go[:, :D])) - out)
        # (the sum's error times what the norm multiplies it with: |out / ref|, and the same number where the sum is 0 and that is 0 / 0)
        most = (np.abs(v) + np.abs(hv)) * (1.0 if pre is None else np.abs(pre)) / np.sqrt((ref * ref).mean(-1, keepdims=True) + eps)
        assert (err <= U32 * 2 * (n + 8) * most + ROUND[qt] * np.abs(out) + TINY[qt] + U32 * np.abs(out) * n).all()
        for a in (gs, go):
            assert (np.ascontiguousarray(a[:, D:]).view(np.uint8) == 0xFF).all()
        # in place, and each output alone
        hb2, xb2 = DevBuf.of(g, h), DevBuf.of(g, x)
        ops.norm_residual(qt, rt, xb2, s, hb2, s, hb2, s, xb2, s, T, D, eps, scale, post=opt(post), gate=opt(gate), pre=opt(pre))
        same = lambda a, b: np.array_equal(np.ascontiguousarray(a[:, :D]).view(np.uint8), np.ascontiguousarray(b[:, :D]).view(np.uint8))  # noqa: E731
        assert same(hb2.read(elt_dtype(rt)).reshape(T, s), gs) and same(xb2.read(elt_dtype(qt)).reshape(T, s), go)
        o.fill(0)
        ops.norm_residual(qt, rt, xb, s, hb, s, None, 0, o, s, T, D, eps, scale, post=opt(post), gate=opt(gate), pre=opt(pre))
        assert same(o.read(elt_dtype(qt)).reshape(T, s), go)
        h1.fill(0)
        ops.norm_residual(qt, rt, xb, s, hb, s, h1, s, None, 0, T, D, eps, scale, post=opt(post), gate=opt(gate), pre=opt(pre))
        assert same(h1.read(elt_dtype(rt)).reshape(T, s), gs)
    # a model's first norm: no block in front of it
    o.fill(0)
    ops.norm_residual(qt, rt, None, 0, hb, s, None, 0, o, s, T, D, eps, pre=DevBuf.of(g, vec[2]))
    near(from_type(qt, np.ascontiguousarray(o.read(elt_dtype(qt)).reshape(T, s)[:, :D])), rms(hv, eps) * vec[2], qt, norm_roundings(D) + 4, "first norm")


def test_norms_of_zeros_and_of_what_is_not_finite(ops):
    """A row of zeros is zeros; a NaN or an infinity stays in its row."""
    g, D = ops.gpu, 256
    y = np.ones((4, D), np.float32)
    y[0] = 0.0
    y[1, 3], y[2, 5] = np.nan, np.inf
    out = DevBuf(g, y.nbytes)
    ops.norm_gated(F32, DevBuf.of(g, y), D, DevBuf.of(g, np.ones_like(y)), D, None, out, D, 4, D, 1, 1e-5)
    got = out.read(np.float32).reshape(4, D)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and not np.isfinite(got[2, 5]) and np.isfinite(got[3]).all()
    ops.norm_residual(F32, F32, DevBuf.of(g, y), D, DevBuf.of(g, np.zeros_like(y)), D, None, 0, out, D, 4, D, 1e-5)
    got = out.read(np.float32).reshape(4, D)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and not np.isfinite(got[2, 5]) and np.isfinite(got[3]).all()


# ---- 4-bit weights

def q4_rule(w, group):
    """The q4_0 rule over groups of a row, in float32 as the header states it: (q, half scales)."""
    M, K = w.shape
    pad = -K % group
    v = np.concatenate([w, np.zeros((M, pad), np.float32)], 1).reshape(M, -1, group)
    i = np.abs(v).argmax(2)
    d = (np.take_along_axis(v, i[..., None], 2)[..., 0] / np.float32(-8.0)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, np.float32(1.0) / d, np.float32(0.0)).astype(np.float32)
    t = (v * inv[..., None]).astype(np.float32) + np.float32(8.5)
    q = np.minimum(15, t.astype(np.int32))
    return q.reshape(M, -1)[:, :K], d.astype(np.float16)


@pytest.mark.parametrize("M,K,group,pad", [(16, 128, 32, 0), (1, 1, 32, 0), (17, 130, 64, 3), (40, 1000, 128, 0), (33, 257, 32, 7), (5, 127, 128, 1), (64, 64, 64, 0)])
def test_q4_pack_floats(ops, M, K, group, pad):
    g = ops.gpu
    w = (np.random.default_rng(M).standard_normal((M, K + pad)) * 0.02).astype(np.float32)
    w[0, :K // 2] = 0.0                                # a group of zeros
    out = DevBuf(g, ops.q4_bytes(M, K, group) + 16)
    out.fill(0xFF)
    ops.q4_pack(0, DevBuf.of(g, w), K + pad, M, K, group, out)
    raw = out.read(np.uint8)
    assert (raw[-16:] == 0xFF).all()
    got, q, s = q4_weights(raw[:-16], M, K, group)
    wq, ws = q4_rule(w[:, :K], group)
    assert np.array_equal(q, wq) and np.array_equal(s.view(np.uint16), np.repeat(ws, group, 1)[:, :K].view(np.uint16))
    # half a step of a group's scale, or a whole one at the far end of the range (15 stands for 7 and more), and the scale's rounding
    assert (np.abs(got - w[:, :K]) <= np.abs(s.astype(np.float64)) * 1.01 + 8 * 2.0 ** -25).all()
    # what lies past M and K is weights of 0
    Mp, Kp = (M + 15) // 16 * 16, (K + 127) // 128 * 128
    full, qf, sf = q4_weights(raw[:-16], Mp, Kp, group)
    assert (full[M:] == 0).all() and (full[:, K:] == 0).all() and (qf[M:] == 8).all() and (qf[:, K:] == 8).all()


def test_q4_pack_blocks(ops):
    """q4_0 blocks as model files hold them, rows with a gap between them."""
    g, M, K, gap = ops.gpu, 19, 160, 10
    r = np.random.default_rng(0)
    rowb = K // 32 * 18
    src = r.integers(0, 256, (M, rowb + gap), dtype=np.uint8)
    scales = (r.standard_normal((M, K // 32)) * 0.02).astype(np.float16)
    blocks = src[:, :rowb].reshape(M, K // 32, 18)
    blocks[:, :, :2] = scales.view(np.uint8).reshape(M, K // 32, 2)
    src[:, :rowb] = blocks.reshape(M, rowb)
    out = DevBuf(g, ops.q4_bytes(M, K, 32))
    ops.q4_pack(1, DevBuf.of(g, src), rowb + gap, M, K, 32, out)
    _, q, s = q4_weights(out.read(np.uint8), M, K, 32)
    n = blocks[:, :, 2:]
    want = np.concatenate([n & 15, n >> 4], 2).reshape(M, K)
    assert np.array_equal(q, want) and np.array_equal(s, np.repeat(scales, 32, 1))


def random_q4(M, K, group, seed):
    r = np.random.default_rng(seed)
    b = r.integers(0, 256, ((M + 15) // 16, (K + 127) // 128, 1024 + 32 * (128 // group)), dtype=np.uint8)
    s = (0.02 * np.exp(0.3 * r.standard_normal(b.shape[:2] + (16 * 128 // group,)))).astype(np.float16)
    b[:, :, 1024:] = s.view(np.uint8)
    return b


def check_product(got, xv, w64, qt, what):
    """The weights are exact; a float32 row's value enters within 2^-21 of itself, or of 2^-36 of its tile's largest; products
    of 11 and 4 bits are exact and their float32 sums round once an addition (K of them at most, the usual error is their
    root), a scale and a tile's power of two once each."""
    ref = xv @ w64.T
    K = xv.shape[1]
    most = np.abs(xv) @ np.abs(w64).T
    big = np.abs(xv).max(1, keepdims=True) if K else 0
    tol = (2.0 ** -21 + U32 * (16 + 4 * K ** 0.5)) * most + 2.0 ** -36 * big * np.abs(w64).sum(1) + ROUND[qt] * np.abs(ref) + TINY[qt]
    err = np.abs(got.astype(np.float64) - ref)
    assert np.isfinite(got).all() and (err <= tol).all(), "%s: %.3g of %.3g" % (what, (err - tol).max(), np.abs(ref).max())


# M, K, T, pads of x and y
PRODUCTS = [(16, 128, 1, 0, 0), (1, 1, 1, 0, 0), (17, 130, 3, 3, 5), (200, 1000, 16, 8, 0), (64, 4096, 1, 0, 0), (48, 8200, 2, 0, 1), (33, 2050, 16, 6, 3), (16, 8192, 8, 0, 0),
            (1000, 257, 5, 1, 0), (2, 70000, 1, 0, 0), (16, 20000, 16, 0, 0), (5, 127, 7, 0, 0), (4097, 64, 9, 0, 7)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("M,K,T,px,py", PRODUCTS)
def test_q4_product(ops, qt, group, M, K, T, px, py):
    g = ops.gpu
    b = random_q4(M, K, group, M + K)
    w64, _, _ = q4_weights(b, M, K, group)
    x, xv = rows(qt, T, K, K + px, 3)
    # (what lies past K in the tiles meets no row's value: values behind a row are not read as its own)
    y = DevBuf(g, T * (M + py) * E[qt])
    y.fill(0xFF)
    ops.q4_product(qt, DevBuf.of(g, x), K + px, DevBuf.of(g, b), group, y, M + py, T, M, K)
    got = y.read(elt_dtype(qt)).reshape(T, M + py)
    check_product(from_type(qt, np.ascontiguousarray(got[:, :M])), xv, w64, qt, (M, K, T))
    assert (np.ascontiguousarray(got[:, M:]).view(np.uint8) == 0xFF).all()


@pytest.mark.parametrize("qt", [F32, BF16])
def test_q4_product_of_large_and_small_rows(ops, qt):
    """Rows far outside a half's range, rows of widely different sizes in one call, a row of zeros, tiles of zeros."""
    g, M, K, T = ops.gpu, 40, 512, 6
    b = random_q4(M, K, 32, 1)
    w64, _, _ = q4_weights(b, M, K, 32)
    x = np.random.default_rng(0).standard_normal((T, K))
    x *= np.array([1e30, 1e-30, 1.0, 0.0, 1e6, 1.0])[:, None]
    x[5, :256] = 0.0
    x[2] *= np.exp(4 * np.random.default_rng(1).standard_normal(K))
    raw, xv = to_type(qt, x)
    y = DevBuf(g, T * M * E[qt])
    ops.q4_product(qt, DevBuf.of(g, raw), K, DevBuf.of(g, b), 32, y, M, T, M, K)
    check_product(from_type(qt, y.read(elt_dtype(qt)).reshape(T, M)), xv.astype(np.float64), w64, qt, "sizes")


@pytest.mark.parametrize("qt", TYPES)
def test_q4_product_keeps_what_is_not_finite_in_its_row(ops, qt):
    g, M, K, T = ops.gpu, 20, 300, 4
    b = random_q4(M, K, 64, 2)
    w64, _, _ = q4_weights(b, M, K, 64)
    x = np.random.default_rng(3).standard_normal((T, K)).astype(np.float32)
    raw, xv = to_type(qt, x)
    y, clean = DevBuf(g, T * M * E[qt]), DevBuf(g, T * M * E[qt])
    wb = DevBuf.of(g, b)
    ops.q4_product(qt, DevBuf.of(g, raw), K, wb, 64, clean, M, T, M, K)
    x[1, 77], x[2, 299] = np.nan, np.inf
    raw, _ = to_type(qt, x)
    ops.q4_product(qt, DevBuf.of(g, raw), K, wb, 64, y, M, T, M, K)
    got, want = (from_type(qt, a.read(elt_dtype(qt)).reshape(T, M)) for a in (y, clean))
    assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any() and np.array_equal(got[[0, 3]], want[[0, 3]])


# ---- a layer

class Model:
    """One state-space layer: residual + norm, in-projection, convolution and scan, gated norm, out-projection, residual + norm."""

    def __init__(self, g, ops, qt, cap):
        self.g, self.ops, self.qt, self.cap = g, ops, qt, cap
        self.D, self.eps = 192, 1e-5
        self.L = L = Layer(4, 32, 64, 2, 4, seed=5)
        self.row = 2 * L.inner + 2 * L.G * L.N + L.H
        r = np.random.default_rng(6)
        f = lambda *s: (1.0 + 0.1 * r.standard_normal(s)).astype(np.float32)  # noqa: E731
        self.pre, self.gn, self.post, self.next = f(self.D), f(L.inner), f(self.D), f(self.D)
        self.win, self.wout = random_q4(self.row, self.D, 32, 7), random_q4(self.D, L.inner, 64, 8)
        of = lambda a: DevBuf.of(g, a)  # noqa: E731
        self.b = {k: of(getattr(self, k)) for k in ("pre", "gn", "post", "next", "win", "wout")}
        self.lw = tuple(of(a) for a in (L.cw, L.cb, L.a, L.dtb, L.d))
        self.ring, self.state = of(np.full((cap, L.chan), np.nan, np.float32)), DevBuf(g, L.H * L.P * L.N * 4)

    def buffers(self, T):
        L, e = self.L, E[self.qt]
        n = {"h": T * self.D * 4, "h1": T * self.D * 4, "x": T * self.D * e, "z": T * self.row * e, "y": T * L.inner * e, "o": T * self.D * e, "n": T * self.D * e,
             "sc": max(4, 4 * self.ops.ssm_prompt_scratch(T, L.H, L.P, L.N, L.G, L.K))}
        return {k: DevBuf(self.g, v) for k, v in n.items()}

    def run(self, b, T, p0, step):
        ops, L, qt, e, D = self.ops, self.L, self.qt, E[self.qt], self.D
        ops.norm_residual(qt, F32, None, 0, b["h"], D, None, 0, b["x"], D, T, D, self.eps, pre=self.b["pre"])
        for t in range(0, T, 16):
            m = min(16, T - t)
            ops.q4_product(qt, b["x"].view(t * D * e, m * D * e), D, self.b["win"], 32, b["z"].view(t * self.row * e, m * self.row * e), self.row, m, self.row, D)
        xbc, dt = b["z"].view(L.inner * e, b["z"].len - L.inner * e), b["z"].view((L.inner + L.chan) * e, b["z"].len - (L.inner + L.chan) * e)
        if step:
            ops.ssm_step(qt, xbc, self.row, dt, self.row, *self.lw, self.ring, self.cap, p0, T, L.H, L.P, L.N, L.G, L.K, self.state, self.state, b["y"], L.inner)
        else:
            ops.ssm_prompt(qt, xbc, self.row, dt, self.row, *self.lw, self.ring, self.cap, p0, T, L.H, L.P, L.N, L.G, L.K, self.state if p0 else None, self.state, b["y"],
                           L.inner, b["sc"])
        ops.norm_gated(qt, b["y"], L.inner, b["z"], self.row, self.b["gn"], b["y"], L.inner, T, L.inner, L.G, self.eps)
        for t in range(0, T, 16):
            m = min(16, T - t)
            ops.q4_product(qt, b["y"].view(t * L.inner * e, m * L.inner * e), L.inner, self.b["wout"], 64, b["o"].view(t * D * e, m * D * e), D, m, D, L.inner)
        ops.norm_residual(qt, F32, b["o"], D, b["h"], D, b["h1"], D, b["n"], D, T, D, self.eps, 0.5, post=self.b["post"], pre=self.b["next"])

    def plain(self, h):
        """The whole run in float64: (the stream behind the layer, the next norm's rows)."""
        L, T = self.L, h.shape[0]
        win, wout = q4_weights(self.win, self.row, self.D, 32)[0], q4_weights(self.wout, self.D, L.inner, 64)[0]
        z = (rms(h, self.eps) * self.pre) @ win.T
        y = scan(L, z[:, L.inner:L.inner + L.chan], z[:, L.inner + L.chan:], np.zeros((3, L.chan)), np.zeros((L.H, L.P, L.N)))[0]
        y = rms((y * silu(z[:, :L.inner])).reshape(T, L.G, -1), self.eps).reshape(T, -1) * self.gn
        s = h + 0.5 * rms(y @ wout.T, self.eps) * self.post
        return s, rms(s, self.eps) * self.next


@pytest.mark.parametrize("qt,rel", [(F32, 2.0 ** -16), (F16, 6 * 2.0 ** -11), (BF16, 6 * 2.0 ** -8)])
def test_a_layer_for_a_prompt_and_its_tokens(ops, qt, rel):
    """A prompt of 70 rows and 6 tokens behind it against the whole layer in float64. (float32 rows: the calls' own errors,
    2^-18 each at most in the mean, four of them in line; 16-bit rows: each of the layer's five row buffers rounds once, and
    a rounding of the projected rows reaches the scan three times.)"""
    m = Model(ops.gpu, ops, qt, 4)
    h = np.random.default_rng(9).standard_normal((76, m.D)).astype(np.float32)
    want, nxt = m.plain(h.astype(np.float64))
    got, gn = [], []
    b = m.buffers(70)
    b["h"].write(h[:70])
    m.run(b, 70, 0, False)
    got.append(b["h1"].read(np.float32).reshape(70, -1))
    gn.append(from_type(qt, b["n"].read(elt_dtype(qt))).reshape(70, -1))
    b = m.buffers(1)
    for t in range(70, 76):
        b["h"].write(h[t])
        m.run(b, 1, t, True)
        got.append(b["h1"].read(np.float32).reshape(1, -1))
        gn.append(from_type(qt, b["n"].read(elt_dtype(qt))).reshape(1, -1))
    for a, r in ((np.concatenate(got), want), (np.concatenate(gn), nxt)):
        assert np.linalg.norm(a - r) <= rel * np.linalg.norm(r), np.linalg.norm(a - r) / np.linalg.norm(r)


@pytest.mark.parametrize("step,T", [(True, 1), (False, 70)])
def test_a_layer_in_a_graph(step, T):
    """The same calls recorded once and replayed, other inputs each time, with the program's own copies, waits and eager calls
    between: each replay gives the eager calls' bits."""
    g = Gpu.open(0)
    ops = Ops(g)
    try:
        m = Model(g, ops, F32, 8)
        b, p0 = m.buffers(T), 40
        start, ring = np.random.default_rng(1).standard_normal(m.state.len // 4).astype(np.float32), np.random.default_rng(2).standard_normal((8, m.L.chan)).astype(np.float32)

        def reset(rep):
            b["h"].write(np.random.default_rng(50 + rep).standard_normal((T, m.D)).astype(np.float32))
            m.state.write(start)
            m.ring.write(ring)
            b["n"].fill(0xFF)
            g.sync()

        outs = lambda: [a.read(np.uint32) for a in (b["h1"], b["n"], m.state, m.ring)]  # noqa: E731
        h = C.c_void_p()
        ops.ok(ops.k.q35_graph_begin(ops.raw(), C.byref(h)), "graph begin")
        try:
            m.run(b, T, p0, step)
        finally:
            ops.ok(ops.k.q35_graph_end(ops.raw(), h), "graph end")
        for rep in range(4):
            reset(rep)
            ops.ok(ops.k.q35_graph_launch(ops.raw(), h), "graph launch")
            got = outs()
            reset(rep)
            m.run(b, T, p0, step)
            assert all(np.array_equal(x, y) for x, y in zip(got, outs())), rep
        ops.k.q35_graph_free(h)
    finally:
        g.close()


def test_wrappers_check_their_buffers(ops):
    g = ops.gpu
    b = DevBuf(g, 1 << 14)
    small = b.view(0, 60)
    for call in (lambda: ops.norm_gated(F32, small, 16, b, 16, None, b, 16, 1, 16, 1, 1e-5), lambda: ops.norm_gated(F32, b, 16, b, 16, small, b, 16, 1, 16, 1, 1e-5),
                 lambda: ops.norm_residual(F32, F32, small, 16, b, 16, b, 16, b, 16, 1, 16, 1e-5), lambda: ops.norm_residual(F32, F32, None, 16, b, 16, b, 16, small, 16, 1, 16, 1e-5),
                 lambda: ops.q4_product(F32, small, 16, b, 32, b, 16, 1, 16, 16), lambda: ops.q4_product(F32, b, 16, small, 32, b, 16, 1, 16, 16),
                 lambda: ops.q4_product(F32, b, 16, b, 32, small, 16, 1, 16, 16), lambda: ops.q4_pack(0, small, 16, 1, 16, 32, b), lambda: ops.q4_pack(0, b, 16, 1, 16, 32, small)):
        with pytest.raises(Error, match="needs"):
            call()
    for call in (lambda: ops.norm_gated(7, b, 16, b, 16, None, b, 16, 1, 16, 1, 1e-5), lambda: ops.norm_residual(3, 0, b, 16, b, 16, b, 16, b, 16, 1, 16, 1e-5),
                 lambda: ops.q4_product(-1, b, 16, b, 32, b, 16, 1, 16, 16)):
        with pytest.raises(Error, match="rows of type"):
            call()


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("M,K", [(40, 4100), (4112, 4096), (1000, 9000)])
def test_a_q4_products_row_alone_and_among_others(ops, qt, group, M, K):
    """A verify pass's rows have the bits of their own tokens' passes, whether the rows' operands fit LDS or not."""
    g, T = ops.gpu, 16
    wb = DevBuf.of(g, random_q4(M, K, group, 3))
    raw, _ = to_type(qt, np.random.default_rng(8).standard_normal((T, K)))
    rows, y = DevBuf.of(g, raw), DevBuf(g, T * M * E[qt])
    whole = None
    for n in (16, 5, 1):
        for t in range(0, T, n):
            m = min(n, T - t)
            ops.q4_product(qt, rows.view(t * K * E[qt], m * K * E[qt]), K, wb, group, y.view(t * M * E[qt], m * M * E[qt]), M, m, M, K)
        got = y.read(np.uint8)
        whole = got if whole is None else whole
        assert np.array_equal(got, whole), n


# lengths about a wave's and a work-group's pieces of 4 and 8 values, whole and not, at every alignment of a row
RAGGED = [63, 65, 67, 253, 257, 509, 513, 4093, 4097, 8191, 8193, 16385, 16387, 32769]


@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("W", RAGGED)
def test_norms_of_ragged_rows(ops, qt, W):
    for order, (T, groups, py, pz, po) in enumerate([(2, 3, 1, 0, 3), (3, 1, 0, 2, 1)]):
        test_norm_gated(ops, qt, order, T, W * groups, groups, py, pz, po)
    test_norm_residual(ops, qt, F32, 2, W, 1)
    test_norm_residual(ops, qt, qt, 3, W, 0)


@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("M,K,T,px,py", [(48, 257, 7, 0, 1), (4112, 1843, 3, 0, 0), (17, 8191, 16, 3, 0), (5, 9, 2, 0, 0)])
def test_q4_product_of_ragged_rows(ops, qt, M, K, T, px, py):
    test_q4_product(ops, qt, 64, M, K, T, px, py)
