"""The operators of a hybrid model's layers (include/ns_layer.h) from their definitions, in float64 and row by row, and how
far a float32 computation of them may be: what the layer tests share."""
import numpy as np

from oracle import orc

F32, F16, BF16 = 0, 1, 2
U32 = 2.0 ** -24
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}      # half a step of the output's type, relative
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}    # half a step among the smallest


def to_type(qt, x):
    """(the array that goes to the GPU, the values it holds as float32)."""
    x = np.ascontiguousarray(x, np.float32)
    if qt == F32:
        return x, x
    b = (orc.f2h if qt == F16 else orc.f2bf)(x)
    return b, (orc.h2f if qt == F16 else orc.bf2f)(b)


def from_type(qt, raw):
    return raw.view(np.float32) if qt == F32 else (orc.h2f if qt == F16 else orc.bf2f)(raw)


def elt_dtype(qt):
    return np.float32 if qt == F32 else np.uint16


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1.0 + np.exp(-v))


class Layer:
    """A state-space layer's weights, random but for its sizes."""

    def __init__(self, H, P, N, G, K, seed, bias=True, rate=None):
        self.H, self.P, self.N, self.G, self.K = H, P, N, G, K
        self.inner, self.chan = H * P, H * P + 2 * G * N
        r = np.random.default_rng(seed)
        f = lambda a: np.ascontiguousarray(a, np.float32)  # noqa: E731
        self.cw = f(r.standard_normal((self.chan, K)) * 0.5)
        self.cb = f(r.standard_normal(self.chan) * 0.1) if bias else None
        self.a = f(-r.uniform(1.0, 16.0, H) if rate is None else np.full(H, rate))
        self.dtb = f(r.uniform(-6.0, -2.0, H)) if bias else None
        self.d = f(1.0 + 0.1 * r.standard_normal(H)) if bias else None


def scan(L, raw, step, past, h0, lo=0.0, hi=np.inf):
    """raw [T][chan], step [T][H], past [K - 1][chan] rows in front of them, h0 [H][P][N]: (y [T][H P], h [T + 1][H][P][N],
    bound [T][H P], hbound [T + 1][H][P][N]) in float64. The bounds are of a float32 computation, to be scaled by an
    error of 2^-24 a rounding: the same sums over absolute values, the convolution's over its taps (|silu(v)| <= |v|)."""
    T = raw.shape[0]
    x64 = np.concatenate([past.astype(np.float64), raw.astype(np.float64)])
    cb = 0.0 if L.cb is None else L.cb.astype(np.float64)
    conv = sum(x64[k:k + T] * L.cw[:, k].astype(np.float64) for k in range(L.K)) + cb
    most = sum(np.abs(x64[k:k + T] * L.cw[:, k]) for k in range(L.K)) + np.abs(cb)
    c = silu(conv)
    dt = np.logaddexp(step.astype(np.float64) + (0.0 if L.dtb is None else L.dtb.astype(np.float64)), 0.0)
    dt = np.where(dt < lo, lo, np.where(dt > hi, hi, dt))
    d = np.zeros(L.H) if L.d is None else L.d.astype(np.float64)
    per = L.H // L.G

    def parts(v):
        grp = lambda s: np.repeat(s.reshape(T, L.G, L.N), per, 1)  # noqa: E731
        return v[:, :L.inner].reshape(T, L.H, L.P), grp(v[:, L.inner:L.inner + L.G * L.N]), grp(v[:, L.inner + L.G * L.N:])

    (x, B, C), (xa, Ba, Ca) = parts(c), parts(most)
    h, hb = np.empty((T + 1, L.H, L.P, L.N)), np.empty((T + 1, L.H, L.P, L.N))
    h[0] = h0
    hb[0] = np.abs(h0)
    y, yb = np.empty((T, L.H, L.P)), np.empty((T, L.H, L.P))
    for t in range(T):
        keep = np.exp(dt[t] * L.a)[:, None, None]
        h[t + 1] = h[t] * keep + (dt[t][:, None] * x[t])[..., None] * B[t][:, None, :]
        hb[t + 1] = hb[t] * keep + (dt[t][:, None] * xa[t])[..., None] * Ba[t][:, None, :]
        y[t] = (h[t + 1] * C[t][:, None, :]).sum(2) + d[:, None] * x[t]
        yb[t] = (hb[t + 1] * Ca[t][:, None, :]).sum(2) + np.abs(d)[:, None] * xa[t]
    return y.reshape(T, L.inner), h, yb.reshape(T, L.inner), hb


def scan_tolerance(T, N):
    """Roundings, of 2^-24 each, between a value of the scan and float32 arithmetic, against sums of absolute values: the
    taps and silu (12) once for each of x, B and C, the step size (8) and what it does to a decay - the exponent's relative
    error times the exponent, at most 1 / e of what is left of a row after it, and an exponential (together 8) - the sums
    over N features (their worst case grows with N, their usual one with its root: 4 sqrt N) and over the rows (one
    multiply-add each, decayed: 4 sqrt T), and operands of a matrix product that hold 21 bits or more (8 each, three of
    them)."""
    return U32 * (36 + 16 + 24 + 4 * N ** 0.5 + 4 * T ** 0.5)


def check_scan(got, ref, bound, qt, T, N, what):
    assert np.isfinite(got).all(), what
    err = np.abs(got.astype(np.float64) - ref)
    tol = scan_tolerance(T, N) * bound + ROUND[qt] * np.abs(ref) + TINY[qt]
    if qt != F32:
        # 16-bit rows: the operands of the products that only reach y may be halfs (three of 2^-11: x, C or the product of
        # B and C with its decay, and the state)
        tol = tol + 3 * 2.0 ** -11 * bound
    at = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), "%s: %s is %.9g, should be %.9g, off by %.3g of %.3g" % (what, at, got[at], ref[at], err[at], tol[at])
    size = np.linalg.norm(ref)
    if size:
        # root mean square: those roundings are of either sign
        rel = np.linalg.norm(err) / size
        assert rel <= 2.0 ** -18 + {F32: 0.0, F16: 2.0 * 2.0 ** -11, BF16: 2.0 ** -8}[qt], "%s: relative error %.3g" % (what, rel)


def rms(v, eps):
    return v / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def q4_weights(w, M, K, group):
    """The tiles' bytes as float64 [M][K], value by value where the header says they are."""
    mt, kt, gr = (M + 15) // 16, (K + 127) // 128, 128 // group
    tile = 1024 + 32 * gr
    w = np.asarray(w, np.uint8).reshape(mt, kt, tile)
    m, k = np.arange(M)[:, None], np.arange(K)[None]
    t = w[m // 16, k // 128]
    i, e = k % 128, k % 8
    at = 16 * (m % 16 + 16 * (i // 8 % 4)) + 4 * (i // 32) + (e % 2) * 2 + e // 4
    byte = np.take_along_axis(t, at[..., None], 2)[..., 0]
    q = np.where(e // 2 % 2 == 0, byte & 15, byte >> 4).astype(np.int64)
    sc = np.ascontiguousarray(w[:, :, 1024:]).view(np.float16).reshape(mt, kt, 16 * gr)
    s = np.take_along_axis(sc[m // 16, k // 128], ((m % 16) // 4 * 4 * gr + i // group * 4 + m % 4)[..., None], 2)[..., 0]
    return (q - 8) * s.astype(np.float64), q, s
