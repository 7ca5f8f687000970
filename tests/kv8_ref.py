"""Caches of 8-bit values in blocks of tokens in numpy, in 64 bits and one sequence after another: what include/ns_kv8.h says, written from
it alone."""
import numpy as np

INT8, E4M3 = 0, 1
F32, F16, BF16 = 0, 1, 2
MOST = {INT8: 127.0, E4M3: 448.0}
HELD = {INT8: (-24, 9), E4M3: (-15, 7)}


def e4m3_values():
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9.0)
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7, -v, v)


E4 = e4m3_values()
_UP = E4[:127]                                            # 0 .. 448, ascending: code i is value i


def values(form, codes):
    """Codes (uint8) as the numbers they are."""
    return codes.view(np.int8).astype(np.float64) if form == INT8 else E4[codes]


def encode(form, x):
    """Numbers in units of their scale -> codes: to nearest, to the even one between two; NaN 0, larger ones the largest."""
    x = np.clip(np.nan_to_num(np.asarray(x, np.float64), nan=0.0), -MOST[form], MOST[form])
    if form == INT8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    hi = np.searchsorted(_UP, a).clip(1, 126)
    lo = hi - 1
    d0, d1 = a - _UP[lo], _UP[hi] - a
    code = np.where((d1 < d0) | ((d1 == d0) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    return np.where(np.signbit(x), code | 0x80, code).astype(np.uint8)


def scale_of(form, x):
    """The least scale that holds x's magnitudes."""
    a = np.abs(np.nan_to_num(x, nan=0.0)).max() if x.size else 0.0
    lo, hi = HELD[form]
    for e in range(lo, hi):
        if a <= 2.0 ** e * MOST[form]:
            return 2.0 ** e
    return 2.0 ** hi


class Cache:
    def __init__(self, form, blocks, Hkv, B, D, seed=0):
        """Pools of anything at all: what no call wrote must not matter. (e4m3: NaN codes among it)"""
        r = np.random.default_rng(seed)
        self.form, self.blocks, self.Hkv, self.B, self.D = form, blocks, Hkv, B, D
        self.k, self.v = (r.integers(0, 256, (blocks, Hkv, B, D)).astype(np.uint8) for _ in range(2))
        self.ks, self.vs = (2.0 ** r.integers(-6, 6, (blocks, Hkv)).astype(np.float32) for _ in range(2))

    def there(self, table, seq, p):
        e = p // self.B
        return e < table.shape[1] and 0 <= table[seq, e] < self.blocks

    def store(self, k, v, table, lens, start, most):
        """k, v [T][Hkv][D] float64 of values as the rows' type holds them."""
        for s in range(len(lens)):
            n = min(start[s + 1] - start[s], most)
            if lens[s] < 0 or n <= 0:
                continue
            p0, p1 = int(lens[s]), int(lens[s]) + int(n)
            for e in range(p0 // self.B, (p1 - 1) // self.B + 1):
                if not self.there(table, s, e * self.B):
                    continue
                b, a, z = table[s, e], max(e * self.B, p0), min((e + 1) * self.B, p1)
                at = slice(a - e * self.B, z - e * self.B)
                for pool, scale, rows in ((self.k, self.ks, k), (self.v, self.vs, v)):
                    for h in range(self.Hkv):
                        x = rows[start[s] + a - p0:start[s] + z - p0, h]
                        s1 = scale_of(self.form, x)
                        if a > e * self.B and scale[b, h] >= s1:
                            s1 = float(scale[b, h])
                        elif a > e * self.B:
                            other = np.ones(self.B, bool)
                            other[at] = False
                            pool[b, h, other] = encode(self.form, values(self.form, pool[b, h, other]) * (float(scale[b, h]) / s1))
                        pool[b, h, at] = encode(self.form, x / s1)
                        scale[b, h] = s1

    def tokens(self, table, seq, n):
        """The first n tokens' keys and values [n][Hkv][D]; zeros where there is no block."""
        k, v = np.zeros((n, self.Hkv, self.D)), np.zeros((n, self.Hkv, self.D))
        for e in range((n + self.B - 1) // self.B):
            if self.there(table, seq, e * self.B):
                b, m = table[seq, e], min(self.B, n - e * self.B)
                for out, pool, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    out[e * self.B:e * self.B + m] = (values(self.form, pool[b, :, :m]) * scale[b].astype(np.float64)[:, None, None]).transpose(1, 0, 2)
        return k, v

    def attend(self, q, table, seq, p0, win=0, scale=0.0, longest=1 << 62):
        """Rows q [T][Hq][D] at tokens p0..: outputs, and the weights given [Hkv][p0 + T]."""
        T, Hq, D = q.shape
        n, G = p0 + T, Hq // self.Hkv
        k, v = self.tokens(table, seq, n)
        out, given = np.zeros((T, Hq, D)), np.zeros((self.Hkv, n))
        pos, key = p0 + np.arange(T)[:, None], np.arange(n)[None]
        seen = (key <= pos) & (key < longest) & ((key > pos - win) if win > 0 else True)
        for h in range(Hq):
            s = np.where(seen, q[:, h] @ k[:, h // G].T * (scale if scale > 0 else D ** -0.5), -np.inf)
            with np.errstate(invalid="ignore", over="ignore"):
                m = s.max(1, keepdims=True)
                w = np.exp(s - np.where(np.isfinite(m), m, 0.0))
                w /= np.where(w.sum(1, keepdims=True) > 0, w.sum(1, keepdims=True), 1.0)
            out[:, h] = w @ v[:, h // G]
            given[h // G] += w.sum(0)
        return out, given

    def give(self, acc0, acc1, table, seq, past, given):
        for t in range(given.shape[1]):
            if self.there(table, seq, t):
                at = (table[seq, t // self.B], slice(None), t % self.B)
                acc1[at] = (acc0[at] if acc0 is not None and t < past else 0.0) + given[:, t]

    def evict(self, acc, table, lens, keep, first, last, to=None, longest=1 << 30):
        """In place, or into the blocks of `to`; the new lengths."""
        new = lens.copy()
        for s, n in enumerate(lens):
            if n < 0 or n > longest:
                continue
            whole = n <= keep
            new[s] = min(n, keep)
            if whole and to is None:
                continue
            dst = table if to is None else to
            moves = []
            for h in range(self.Hkv):
                a = np.array([acc[table[s, t // self.B], h, t % self.B] if self.there(table, s, t) else 0.0 for t in range(n)])
                sure = (np.arange(n) < first) | (np.arange(n) >= n - last)
                order = np.lexsort((np.arange(n), -np.where(a > 0, a, 0.0), ~sure))
                moves.append(np.sort(order[:new[s]]))
            old = [x.copy() for x in (self.k, self.v, self.ks, self.vs, acc)]
            for h in range(self.Hkv):
                for j in range((new[s] + self.B - 1) // self.B):
                    rows = moves[h][j * self.B:(j + 1) * self.B]
                    if not self.there(dst, s, j * self.B) or (to is None and np.array_equal(rows, j * self.B + np.arange(len(rows)))):
                        continue
                    d = dst[s, j]
                    for pool, scale, pool0, scale0 in ((self.k, self.ks, old[0], old[2]), (self.v, self.vs, old[1], old[3])):
                        sc = [float(scale0[table[s, t // self.B], h]) if self.there(table, s, t) else 0.0 for t in rows]
                        s1 = max([2.0 ** HELD[self.form][0]] + sc)
                        for i, t in enumerate(rows):
                            there = self.there(table, s, t)
                            x = values(self.form, pool0[table[s, t // self.B], h, t % self.B]) if there else np.zeros(self.D)
                            pool[d, h, i] = pool0[table[s, t // self.B], h, t % self.B] if there and sc[i] == s1 else encode(self.form, x * (sc[i] / s1))
                        scale[d, h] = s1
                    for i, t in enumerate(rows):
                        acc[d, h, i] = old[4][table[s, t // self.B], h, t % self.B] if self.there(table, s, t) else 0.0
        return new


def same_codes(form, a, b):
    """Equal as numbers (zeros of either sign alike); NaN codes where NaN codes are."""
    return np.array_equal(values(form, a), values(form, b), equal_nan=True)


def to_type(qt, x):
    """float64 -> (what goes to the GPU, the values it stands for)."""
    x = np.asarray(x, np.float32)
    if qt == F32:
        return x, x.astype(np.float64)
    if qt == F16:
        h = x.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(x), np.uint16(0x7FC0), r)
    return r, (r.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def from_type(qt, raw):
    if qt == F32:
        return raw.astype(np.float64)
    if qt == F16:
        return raw.view(np.float16).astype(np.float64)
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def tolerance(qt, ref, reach, vmax, D, n):
    """(absolute, relative L2) for rows against the closed form. reach: the largest sum of |q k| scale log2 e of a row and a token. A score carries 22
    bits of each product and a sum of D of them in float32, an exponential's and a weight's roundings 2^-22 and 2^-23; a weighted mean of values up to
    vmax moves by twice the largest relative error of a weight, and its own sum over n tokens in steps of 32 by a rounding each.
    In the mean these add as squares: sqrt(D) of them for a score of the scale sqrt(mean) ~ 3, far below 2^-17.
    Beside rows of 16 bits a weight's numerator is a half, not its sum: out = sum w (1 + d) v / sum w, |d| <= 2^-11, moves by vmax 2^-11 at most; weights
    under 2^-21 of the row's largest, d up to a half's least step against them, 2^-25 of 2^7 x the largest: by n 2^-32 vmax at most. In the mean d's
    signs are as random as v's: sqrt(sum (w d v)^2) <= 2^-11 sqrt(sum (w v)^2), which is 2^-11 of what the output comes to."""
    weight = np.log(2.0) * reach * (2.0 ** -22 + D * 2.0 ** -24) + 2.0 ** -21
    half = 0.0 if qt == F32 else 2.0 ** -11
    return (vmax * (2 * weight + (n / 32 + 8) * 2.0 ** -24 + half + (n * 2.0 ** -32 if half else 0.0)) + ROUND[qt] * np.abs(ref).max() +
            (2.0 ** -25 if qt == F16 else 0.0), 2.0 ** -17 + half + ROUND[qt])
