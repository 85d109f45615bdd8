"""MXFP4 and the 8-bit paged cache restated in numpy float64, from their definitions:
the expected values of the GPU tests."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _e4m3_table():
    """The value of every e4m3 code byte: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, (b & 7) / 8.0
    v = np.where(e == 0, m * 2.0 ** -6, (1 + m) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


E4M3 = _e4m3_table()


def nearest(x, grid):
    """Index into the ascending ``grid`` nearest to each |x|, ties to the even index,
    saturating at the last (NaN: the last)."""
    a = np.abs(x)
    mid = (grid[1:] + grid[:-1]) / 2
    lo = np.searchsorted(mid, a, side="left")  # a <= mid[lo]: at or below this midpoint
    tie = (lo < len(mid)) & (a == mid[np.minimum(lo, len(mid) - 1)])
    return lo + (tie & (lo % 2 == 1))


# ---------------------------------------------------------------- MXFP4


def mx_quantize(x):
    """(codes uint8 [rows, k], scale bytes uint8 [rows, k / 32]), one code an entry."""
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    b = x.reshape(rows, k // 32, 32)
    a = np.abs(b).max(-1)
    bad = ~np.isfinite(a)
    _, e = np.frexp(np.where(bad, 1.0, a))
    e = np.where(a == 0, -127, np.maximum(e - 1 - 2, -127))
    with np.errstate(invalid="ignore"):
        mag = nearest(np.where(bad[..., None], 0.0, b) * 2.0 ** (-e[..., None].astype(float)), E2M1)
    codes = (mag + 8 * np.signbit(b)).astype(np.uint8)
    return codes.reshape(rows, k), np.where(bad, 255, e + 127).astype(np.uint8)


def mx_values(codes, scales):
    """float64 [rows, k] of one-code-an-entry codes and by-row scale bytes."""
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(float) - 127))
    return v * np.repeat(s, 32, axis=1)


def mx_unpack(packed):
    """One code an entry of codes packed two a byte, the even column low."""
    packed = np.asarray(packed)
    return np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)


# ---------------------------------------------------------------- the cache


def kv_scale(amax):
    """The least 2^e, -60 <= e <= 60, with amax <= 448 * 2^e."""
    e = -60
    while e < 60 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def e4m3_encode(x):
    """e4m3 code bytes of x, saturating at +-448, NaN to 0x7F."""
    x = np.asarray(x, np.float64)
    mag = nearest(np.where(np.isnan(x), 0.0, x), E4M3[:127])
    return np.where(np.isnan(x), 127, mag + 128 * np.signbit(x)).astype(np.uint8)


class Cache:
    """k, v code bytes [pages, heads, block, d] (V by token here), scales [pages, heads]."""

    def __init__(self, pages, heads, d, block):
        self.k = np.zeros((pages, heads, block, d), np.uint8)
        self.v = np.zeros((pages, heads, block, d), np.uint8)
        self.ks = np.ones((pages, heads))
        self.vs = np.ones((pages, heads))
        self.block = block

    def write(self, k, v, table, filled, counts):
        """Rows of sequence b at positions filled[b] onward, ``counts[b]`` of them."""
        pages, heads, blk, _ = self.k.shape
        r = 0
        for b, n in enumerate(counts):
            p, end = filled[b], filled[b] + n
            while p < end:
                slot, m = p % blk, min(blk - p % blk, end - p)
                row, p = r, p + m
                r += m
                at = (p - m) // blk
                page = table[b][at] if at < len(table[b]) else -1
                if not 0 <= page < pages:
                    continue
                for h in range(heads):
                    for code, sc, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
                        y = np.asarray(x[row:row + m, h], np.float64)
                        fin = np.abs(y[np.isfinite(y)])
                        s = kv_scale(fin.max() if fin.size else 0.0)
                        if slot:
                            s = max(s, sc[page, h])
                            if s > sc[page, h]:
                                held = E4M3[code[page, h, :slot]] * (sc[page, h] / s)
                                code[page, h, :slot] = e4m3_encode(held)
                        sc[page, h] = s
                        code[page, h, slot:slot + m] = e4m3_encode(y / s)

    def tokens(self, table_row, n):
        """(k, v) float64 [n, heads, d] and whether each token has a page."""
        pages, heads, blk, d = self.k.shape
        k, v, have = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros(n, bool)
        for p in range(n):
            page = table_row[p // blk] if p // blk < len(table_row) else -1
            if 0 <= page < pages:
                have[p] = True
                k[p] = E4M3[self.k[page, :, p % blk]] * self.ks[page][:, None]
                v[p] = E4M3[self.v[page, :, p % blk]] * self.vs[page][:, None]
        return k, v, have


def attention(q, k, v, have, causal, window, scale):
    """One sequence: q [n, hq, d], k and v [len, heads, d] -> (out, lse, bound). A row sees
    only the tokens it may: nothing of the others enters, NaN or not. bound [n, hq, d] is
    what a result may differ by before its own rounding: float16 weights (2^-11 each), and
    float32 scores, whose error grows with the sum of |q k| (d terms) and with |t| itself."""
    n, hq, d = q.shape
    length, heads, _ = k.shape
    out, lse, bound = np.zeros((n, hq, d)), np.full((n, hq), -np.inf), np.zeros((n, hq, d))
    for i in range(n):
        p = length - n + i
        j = np.arange(length)
        see = have.copy()
        if causal:
            see &= j <= p
        if window:
            see &= j > p - window
        if not see.any():
            continue
        for h in range(hq):
            kk, vv = k[see, h * heads // hq], v[see, h * heads // hq]
            s = kk @ q[i, h] * scale
            m = s.max()
            w = np.exp(s - m)
            out[i, h] = w @ vv / w.sum()
            lse[i, h] = m + np.log(w.sum())
            ds = 2.0 ** -23 * (np.abs(kk) @ np.abs(q[i, h]) * scale * 4 + np.abs(s).max() * 4 + 90)
            rel = 2.0 ** -11 + 2 * ds.max()
            bound[i, h] = rel * (w @ np.abs(vv) / w.sum())
    return out, lse, bound
