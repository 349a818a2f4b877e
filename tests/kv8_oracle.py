"""Plain 64-bit restatements of the 8-bit K/V cache's operators and of the
rotary positions with axes (include/surge.h), for the tests. The quantiser is
computed exactly, in fractions where a rounding is close."""
import numpy as np

LIMIT = 65520.0             # the first magnitude that f16 rounds to infinity


def key_at(r, d):
    return (d // 64) * 1024 + (d // 16 % 4) * 256 + r * 16 + d % 16


def val_at(r, d):
    return (d // 64) * 1024 + (r // 4) * 256 + (d % 16) * 16 + (d // 16 % 4) * 4 + r % 4


class Cache:
    """A cache of `cap` positions: the two buffers as the library lays them out."""

    def __init__(self, nkv, hd, block, cap, rng=None):
        self.nkv, self.hd, self.block = nkv, hd, block
        nt, nb = -(-cap // 16), -(-cap // block)
        self.codes = np.zeros((nt, nkv, 2, 16 * hd), np.int8)
        self.scales = np.zeros((nb, nkv, 2), np.float32)
        if rng is not None:         # what an earlier sequence left
            self.codes[...] = rng.integers(-127, 128, self.codes.shape)
            self.scales[...] = rng.uniform(0.001, 0.1, self.scales.shape)
        r, d = np.meshgrid(np.arange(16), np.arange(hd), indexing="ij")
        self.at = (key_at(r, d), val_at(r, d))

    def rows(self, half, lo, hi):
        """Codes [hi - lo][nkv][hd]."""
        t0, t1 = lo // 16, -(-hi // 16)
        c = self.codes[t0:t1, :, half][:, :, self.at[half]]           # [t][nkv][16][hd]
        return c.transpose(0, 2, 1, 3).reshape(-1, self.nkv, self.hd)[lo - 16 * t0:hi - 16 * t0]

    def put(self, half, lo, codes):
        for i, row in enumerate(codes):
            p = lo + i
            for h in range(self.nkv):
                self.codes[p // 16, h, half][self.at[half][p % 16]] = row[h]

    def values(self, half, n):
        b = np.arange(n) // self.block
        return self.rows(half, 0, n).astype(np.float64) * self.scales[b, :, half].astype(np.float64)[:, :, None]

    def store(self, k, v, base):
        """k, v f32 [n][nkv][hd]."""
        n = len(k)
        for half, x in enumerate((k, v)):
            for b in range(base // self.block, -(-(base + n) // self.block)):
                lo, hi = max(base, b * self.block), min(base + n, (b + 1) * self.block)
                kept = lo - b * self.block
                for h in range(self.nkv):
                    rows = x[lo - base:hi - base, h]
                    was = self.scales[b, h, half] if kept else np.float32(0)
                    mx = np.abs(rows).max()
                    if not mx < LIMIT or np.isnan(was):
                        self.scales[b, h, half] = np.nan
                        new = np.zeros(rows.shape, np.int64)
                    else:
                        s = max(np.float32(mx) * (np.float32(1) / np.float32(127)), was)
                        self.scales[b, h, half] = s
                        new = nearest(rows, s)
                        if kept and s > was:
                            old = self.rows(half, b * self.block, lo)[:, h].astype(np.float64)
                            old = np.rint(old * np.float64(was) / np.float64(s))
                            for i in range(kept):
                                self.codes[(b * self.block + i) // 16, h, half][self.at[half][(b * self.block + i) % 16]] = old[i]
                    for i in range(hi - lo):
                        self.codes[(lo + i) // 16, h, half][self.at[half][(lo + i) % 16]] = new[i]


def nearest(x, s):
    """x / s to the nearest integer, ties to even, |.| <= 127. The quotient of two f32
    numbers is either a tie exactly or further from one than 64 bits resolve."""
    if s == 0:
        return np.zeros(x.shape, np.int64)
    return np.clip(np.rint(x.astype(np.float64) / np.float64(s)), -127, 127).astype(np.int64)


def attention(q, cache, base, scale):
    """q [n][nh][hd] -> (out f64 [n][nh][hd], bound [n][nh][1]): token t over positions 0 .. base + t.

    The bound, with u = 2^-24: a score is exact up to q's rounding (a unit of 2^-23 of the
    head's largest element in every dim) and 8 f32 roundings of its size and of the
    maximum it is taken from; exp adds 2u; p s_V in two halves 4u; sums over n keys add at
    most n / 16 + 64 roundings (16 at a time in the matrix instruction, then one addition
    each). The error of a weight counts twice, in the sum above and in the one below."""
    n, nh, hd = q.shape
    g = nh // cache.nkv
    k, v = cache.values(0, base + n), cache.values(1, base + n)
    out, bound = np.zeros(q.shape), np.zeros((n, nh, 1))
    u = 2.0 ** -24
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(n):
            m = base + t + 1
            for h in range(nh):
                kk, vv, qq = k[:m, h // g], v[:m, h // g], q[t, h].astype(np.float64)
                s = kk @ qq * scale
                p = np.exp(s - s.max())
                out[t, h] = p @ vv / p.sum()
                ds = abs(scale) * 2 * u * np.abs(qq).max() * np.abs(kk).sum(1).max() + 16 * u * np.abs(s).max()
                bound[t, h] = (2 * (ds + 6 * u) + (m / 16 + 64) * u) * np.abs(vv).max()
    return out, bound


def axes_of(rope_dim, sections, order):
    out = []
    for i in range(rope_dim // 2):
        if order:
            out.append(i % 3 if i % 3 and i < 3 * sections[i % 3] else 0)
        else:
            out.append(0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2)
    return out


def rope_axes(x, pos, rope_dim, sections, order, theta):
    """x [n][heads][hd], pos [3][n] -> (out f64, bound): cos and sin are rounded to f32 (half
    a step each), then two products and a sum."""
    half = rope_dim // 2
    out = x.astype(np.float64).copy()
    bound = np.zeros(x.shape)
    for i, a in enumerate(axes_of(rope_dim, sections, order)):
        w = (pos[a].astype(np.float64) * float(np.float32(theta)) ** (-2.0 * i / rope_dim))[:, None]
        lo, hi = x[:, :, i].astype(np.float64), x[:, :, i + half].astype(np.float64)
        out[:, :, i] = lo * np.cos(w) - hi * np.sin(w)
        out[:, :, i + half] = hi * np.cos(w) + lo * np.sin(w)
        bound[:, :, i] = bound[:, :, i + half] = (np.abs(lo) + np.abs(hi)) * 3.1 * 2.0 ** -24
    return out, bound
