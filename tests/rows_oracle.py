"""Plain 64-bit forms of the row operators (norm, rotation, block-scaled append) and of the decode over a
block-scaled cache, in numpy, with bounds on how far a correctly rounded fp32 computation may be from them."""
import numpy as np

D = 128
E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -32, 8


def norm(x, w, eps):
    """x [..., 128] float64."""
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rotate(x, positions, inv_freq, axes=None, interleaved=False, scale=1.0):
    """x [tokens, heads, 128], positions [axes, tokens]; also the magnitude of each element's pair."""
    half = len(inv_freq)
    axes = np.zeros(half, int) if axes is None else np.asarray(axes)
    # the angle as a reduced fraction of a turn in extended precision: far positions lose nothing here either
    turns = np.asarray(positions, np.longdouble)[axes].T * (np.asarray(inv_freq, np.longdouble) / (2 * np.longdouble(np.pi)
                                                            + np.longdouble(2.4492935982947064e-16)))
    angle = ((turns - np.floor(turns)) * 2).astype(np.float64) * np.pi
    c, s = scale * np.cos(angle)[:, None], scale * np.sin(angle)[:, None]
    y, size = x.copy(), np.abs(x)
    lo, hi = (np.s_[..., 0:2 * half:2], np.s_[..., 1:2 * half:2]) if interleaved else (np.s_[..., :half], np.s_[..., half:2 * half])
    y[lo], y[hi] = x[lo] * c - x[hi] * s, x[hi] * c + x[lo] * s
    size[lo] = size[hi] = abs(scale) * (np.abs(x[lo]) + np.abs(x[hi]))
    return y, size


def rows_bound(y, size, eps_type, tiny):
    """Half a step of the output type, and fp32: the norm (128-term sum, rsqrt, two products: < 12 roundings that do not
    average out), the angle's fraction (2^-25 turns-pairs = pi 2^-25) with sincospi (2 steps), two products and a
    sum: fewer than 24 steps of 2^-24 of the pair's size."""
    return eps_type / 2 * np.abs(y) + 24 * 2.0 ** -24 * size + tiny


def e4m3_values():
    """All finite non-negative values, ascending."""
    v = [m * 2.0 ** -9 for m in range(8)]
    for e in range(1, 16):
        v += [(1 + m / 8) * 2.0 ** (e - 7) for m in range(8) if not (e == 15 and m == 7)]
    return np.array(v)


def e4m3_bound(y, scale):
    """Half a step of e4m3 at |y| / scale (2^-4 relative while normal, 2^-10 below), in the units of y."""
    a = np.minimum(np.abs(y) / scale, E4M3_MAX)
    return np.maximum(a * 2.0 ** -4, 2.0 ** -10) * scale


def decode_e4m3(b):
    """Bytes -> float64 (NaN for 0x7f / 0xff)."""
    b = np.asarray(b, np.uint8)
    v = np.append(e4m3_values(), np.nan)[b & 0x7f]
    return np.where(b & 0x80, -v, v)


def round_e4m3(x):
    """Non-negative values below 448 to the nearest one, ties to the even mantissa (its index in the table)."""
    table = e4m3_values()
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    lo = hi - 1
    down, up = x - table[lo], table[hi] - x
    return table[np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)]


def block_tokens(page_size):
    return min(16, page_size & -page_size)


def need_scale(top):
    """Smallest power of two in range with top / scale <= 448."""
    e = MIN_EXP
    while e < MAX_EXP and top > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


class BlockPool:
    """One of K, V: values as appended (exact), scales, and how far each stored value may be off; `slack`: what the bytes of
    slots that no append has reached stand for, in units of the scale (a block whose scale grows is re-encoded whole)."""

    def __init__(self, num_pages, hkv, page_size, slack=0x11):
        self.ps, self.b = page_size, block_tokens(page_size)
        self.x = np.zeros((num_pages, hkv, page_size, D))
        self.off = np.zeros_like(self.x)
        self.slack = np.full(self.x.shape[:3], float(decode_e4m3(slack)))
        self.scale = np.zeros((num_pages, hkv, page_size // self.b))

    def append(self, table, start, y, err):
        """y [n, hkv, 128] at positions start..., err the bound of its fp32 computation."""
        n, at = len(y), 0
        while at < n:
            pos = start + at
            page, off = table[pos // self.ps], pos % self.ps
            inside = off % self.b
            m = min(self.b - inside, n - at)
            blk, first = off // self.b, off - inside
            for h in range(y.shape[1]):
                new = y[at:at + m, h]
                s = need_scale(np.abs(new).max())
                old = self.scale[page, h, blk] if inside else 0.0
                if old > s:
                    s = old
                if inside and s > old:      # re-encoded: exact but for the subnormals of the new scale
                    self.off[page, h, first:off] += 2.0 ** -10 * s
                    self.slack[page, h, first:first + self.b] = round_e4m3(self.slack[page, h, first:first + self.b] * old / s)
                self.scale[page, h, blk] = s
                self.x[page, h, off:off + m] = new
                self.off[page, h, off:off + m] = e4m3_bound(new, s) + 1.07 * err[at:at + m, h]
            at += m


def attention(q, k, v, sm_scale):
    """q [hq, 128], k / v [n, hkv, 128] in float64: (out, bound).

    The kernel's weights are rounded to fp16 (2^-11 each) and the result too; scores are fp32 sums of 128 exact
    products (fewer than 128 steps of 2^-24 of the absolute sum), and exponents of up to ~2^6 are rounded to 2^-19."""
    hq, hkv = q.shape[0], k.shape[1]
    g = hq // hkv
    out, tol = np.zeros((hq, D)), np.zeros((hq, D))
    for h in range(hq):
        kk, vv = k[:, h // g], v[:, h // g]
        s = kk @ q[h] * sm_scale
        p = np.exp(s - s.max())
        p /= p.sum()
        size = p @ np.abs(vv)
        score_err = 128 * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[h])).max() * sm_scale + 2.0 ** -17
        out[h] = p @ vv
        tol[h] = size * (2.0 ** -11 + 2 * score_err) + 2.0 ** -11 * np.abs(out[h]) + 2.0 ** -25
    return out, tol
