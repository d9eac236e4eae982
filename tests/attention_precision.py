"""How near to its definition attention over shared positions has to be on ordinary numbers, and what it does with its
operands' bits, in numpy: so that the tests can leave a part of it out and see that the limits notice.

The limits are for q of a deviation of 2, keys and values of 1 and a scale of 1/8. The 64 products of a score then
have magnitudes that add up to about 10, and the sums after each of the four matrix instructions that make it (16 of the dims
each) are 5 at most, nearly always. An instruction cuts its sum off to 24 bits: by 2^-23 of it at most. If all four
cuts were as large as that, a score would be off by 4 * 5 * 2^-23 = 2.4e-6, and so would its weight, relatively. Over a row
the errors of the weights are as the cuts are (uniform: 1/sqrt(3) of the most, 1.4e-6), and what they have in common drops out of the
quotient, so the row is off by less than that, relative to its 2-norm. Rounding the query's scaling, the exponential (2
ulps), the products with the values, each step's sum and the quotient adds 2^-24 of the row each, in no common
direction: less than 5 * 2^-24 = 3e-7 together with 24 steps in sequence. Over 8-bit pages a query is held to 2^-24 of its largest
element (three times the others), a score to 64 of those: sqrt(64) * 6 * 2^-24 / 8 = 4e-7; a weight times its scale to 2^-23 of
the step's largest. Both are below what the cuts are. Hence 2e-6 over all rows, and three times that for a single one,
of which the scores or their cuts may be twice the usual ones and add up."""
import numpy as np

ALL_ROWS, ONE_ROW = 2e-6, 6e-6
# products of terms (of a page's number, of the query's or the weight's), the largest first
PRODUCTS = {"f32": [(0, 0), (0, 1), (1, 0), (1, 1), (2, 0), (0, 2)], "bf16": [(0, 0), (0, 1), (0, 2)]}


def off(got, want):
    """The 2-norm of got - want, relative to that of want: over all rows, and the largest of a row."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    d, w = np.linalg.norm(got - want, axis=-1), np.linalg.norm(want, axis=-1)
    return np.linalg.norm(d) / np.linalg.norm(w), (d / np.where(w > 0, w, 1.0)).max()


def near(got, want):
    a, b = off(got, want)
    return a <= ALL_ROWS and b <= ONE_ROW


def terms(x):
    """The three bf16 terms of float32 numbers, the largest first (64 bits)."""
    out, x = [], np.asarray(x, np.float32)
    for _ in range(3):
        t = (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        out.append(t.astype(np.float64))
        x = (x - t).astype(np.float32)
    return out


def _sum(page, other, products):
    a, b = (terms(page), terms(other))
    return sum(a[i] @ b[j] for i, j in products)


def row(q, k, v, scale, scores=PRODUCTS["f32"], values=PRODUCTS["f32"]):
    """Attention of q [64] over k, v [n, 64], of those products of terms only; sums in 64 bits."""
    t = _sum(k, (q.astype(np.float32) * np.float32(scale)), scores)
    p = (np.exp(t - t.max())).astype(np.float32)
    return _sum(v.T, p, values) / p.astype(np.float64).sum()


def row_q8(q, k, ks, v, vs, scale, q_bits=24, w_bits=23):
    """The same over levels and scales: the query in so many bits of its largest element, the weights of 32 keys times their
    values' scales in so many of theirs."""
    def held(x, bits):
        unit = 2.0 ** (np.floor(np.log2(np.abs(x).max())) + 2 - bits)
        return np.rint(x / unit) * unit

    t = (k.astype(np.float64) @ held(q.astype(np.float64) * scale, q_bits)) * ks
    p = np.exp(t - t.max())
    o = np.zeros(64)
    for i in range(0, len(k), 32):
        o += held(p[i:i + 32] * vs[i:i + 32], w_bits) @ v[i:i + 32].astype(np.float64)
    return o / p.sum()


def exact(q, k, v, scale):
    t = scale * (k.astype(np.float64) @ q.astype(np.float64))
    p = np.exp(t - t.max())
    return (p / p.sum()) @ v.astype(np.float64)
