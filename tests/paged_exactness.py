# SPDX-License-Identifier: MPL-2.0
"""How far attention over pages in fp32 may be off on average, for inputs without a pattern, and the kernel's arithmetic on the
CPU with products left out, which that bound has to tell from the whole ones.

The bound of a row's elements that holds for any input adds every rounding at its largest; roundings of inputs without a pattern
add up like a random walk, some sqrt(n) times less."""
import numpy as np

U32 = 2.0 ** -24


def deviation(q, k, v, scale):
    """The root of the mean square of one row's error in each output element, in 64 bits: q [HD], k and v [n][HD].

    A score: at most 4 roundings for 16 dimensions of each of the six products, 1.5 HD in all, of partial sums that grow like
    a random walk's: each U32 / sqrt(3) of them in the mean, so HD / 4 times the products' squares; the scale's, the argument's
    and the exponential's, 2 units of the score and 2 of the weight.  A score's error moves a row by its weight times the
    value's distance from the row.  The scale's rounding moves all scores alike.  The sums over the keys are such walks too:
    n / 4 times the squares of their terms; the weights' sum and the quotient a few units of the row."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    n, HD = k.shape
    sc = k @ q * scale
    p = np.exp(sc - sc.max())
    p /= p.sum()
    out = p @ v
    score = HD / 4 * scale * scale * ((k * q) ** 2).sum(1) + 4 * sc * sc + 4
    apart = (v - out) ** 2
    alike = (p * (sc - p @ sc)) @ (v - out)
    return U32 * np.sqrt((p * p * score) @ apart + 4 * alike * alike + n / 4 * (p * p) @ (v * v) + (n / 96 + 6) * out * out)


def terms(x):
    """The three terms of 8 bits, whose sum is x: the upper half, what is left of it to the nearest, and the rest."""
    out, rest = [], np.asarray(x, np.float32)
    for i in range(3):
        u = rest.view(np.uint32).astype(np.uint64)
        t = ((u + (0x7FFF + ((u >> 16) & 1) if i == 1 else 0)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
        out.append(t)
        rest = (rest - t).astype(np.float32)
    assert not rest.any()
    return out


SIX = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]


def sums(a, b, products):
    """a [m][n] by b [n][w] in terms: 16 of the sum at a time, each product of terms added in fp32."""
    a, b = [t.astype(np.float64) for t in terms(a)], [t.astype(np.float64) for t in terms(b)]
    acc = np.zeros((a[0].shape[0], b[0].shape[1]), np.float32)
    for s in range(0, a[0].shape[1], 16):
        for i, j in products:
            acc = (acc + a[i][:, s:s + 16] @ b[j][s:s + 16]).astype(np.float32)
    return acc


def emulated(q, k, v, scale, of_scores=SIX, of_values=SIX):
    """One row as the kernel computes it, with the products of terms that are listed."""
    sc = sums(k, q[:, None], of_scores)[:, 0]
    scale2 = np.float32(abs(scale) * 1.4426950408889634)
    m = np.float32(sc.max() * scale2)
    p = np.exp2((sc.astype(np.float64) * scale2 - m).astype(np.float32)).astype(np.float32)
    return sums(p[None], v, of_values)[0] / np.float32(p.sum(dtype=np.float32))


def last_bits(rng, rows, keys, HD, in_key):
    """Rows and keys whose scores are the last 8 bits of numbers, 0 .. 2 in steps of 2^-7: (x, y) . (1, -1) 2^16, where y is x
    without them, in two dimensions; x is the key's (in_key 1) or the row's.  Key 0 has a score of 0."""
    many, fix = np.zeros((keys if in_key else rows, HD), np.float32), np.zeros((rows if in_key else keys, HD), np.float32)
    x = (1 + rng.integers(0, 1 << 23, len(many)).astype(np.float32) * np.float32(2.0 ** -23)).astype(np.float32)
    d0, d1 = rng.permutation(HD)[:2]
    many[:, d0], many[:, d1] = x, (x.view(np.uint32) & np.uint32(0xFFFFFF00)).view(np.float32)
    fix[:, d0], fix[:, d1] = 2.0 ** 16, -2.0 ** 16
    q, k = (fix, many) if in_key else (many, fix)
    k[0] = 0
    v = rng.choice(np.float32([-1, 1]), (keys, HD))
    return q, k, v


def last_bits_off(q, k, v, got):
    """The largest error of such a row in what it may be.  A score's terms and all their sums are multiples of 2^-7 under 2^17, which
    fp32 holds exactly; so only the exponent (a score up to 2, 4 units), the exponential (2) and a rounding a key in each of
    the sums, 64 where partial sums are joined, are left."""
    sc = k.astype(np.float64) @ q.astype(np.float64)
    p = np.exp(sc)
    off = 2 * (4 * 2 + 2 + len(p) + 64) * U32
    return np.abs(got - p @ v.astype(np.float64) / p.sum()).max() / off
