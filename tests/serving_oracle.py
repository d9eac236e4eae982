"""64-bit definitions of the 8-bit cache, attention over shared positions and 4-bit weights, for the tests
(numpy, CPU)."""
import numpy as np

from ops_oracle import D, PAGE

EPS = 2.0 ** -24


def levels(x, most, scale_type=np.float32, round_scale=None):
    """Levels and scale (float32) of the last axis of x."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(-1)
    with np.errstate(all="ignore"):
        scale = (top.astype(np.float64) / most).astype(np.float32)
        if round_scale is not None:
            scale = round_scale(scale)
        odd = ~np.isfinite(top)
        s = scale.astype(np.float64)[..., None]
        q = np.where((s > 0) & np.isfinite(s), np.rint(x.astype(np.float64) / np.where(s > 0, s, 1.0)), 0.0)
    q = np.where(odd[..., None], 0.0, np.clip(q, -most, most))
    return q.astype(np.int64), np.where(odd, np.float32(np.nan), scale)


def store_q8(k, slots, pages, scales):
    """pages (int8 [P, 16, H * 64]) and scales [P, H, 16] after rows k [rows, H * 64] went into their slots."""
    pages, scales = pages.copy(), scales.copy()
    heads = scales.shape[1]
    q, s = levels(k.reshape(len(k), heads, D), 127)
    for r, slot in enumerate(slots):
        if 0 <= slot < pages.shape[0] * PAGE:
            pages[slot // PAGE, slot % PAGE] = q[r].reshape(-1)
            scales[slot // PAGE, :, slot % PAGE] = s[r]
    return pages, scales


def bf16(x):
    """float32 rounded to nearest-even bf16, as float32."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000
    return np.where(np.isnan(x), np.float32(np.nan), u.astype(np.uint32).view(np.float32))


def quantize_q4(w, group):
    """Levels [n, k] and scales [n, ceil(k / group)] (bf16 values) of weights w."""
    n, k = w.shape
    g = -(-k // group)
    x = np.zeros((n, g * group), np.float32)
    x[:, :k] = w
    q, s = levels(x.reshape(n, g, group), 7, round_scale=bf16)
    return q.reshape(n, -1)[:, :k], s


def pack_q4(q):
    """Levels as bytes: word 4 t + j of a block of 128 holds weights 32 j + 8 t + i at bits 4 i."""
    n, k = q.shape
    blocks = -(-k // 128)
    out = np.zeros((n, blocks, 16), np.uint32)
    for c in range(blocks * 128):
        b, r = divmod(c, 128)
        j, t, i = r // 32, r % 32 // 8, r % 8
        u = (q[:, c] + 8 if c < k else np.full(n, 8)).astype(np.uint32)
        out[:, b, 4 * t + j] |= u << np.uint32(4 * i)
    return out.view(np.uint8).reshape(n, blocks * 64)


def weights(q, scales, group):
    with np.errstate(invalid="ignore"):
        return q * np.repeat(scales.astype(np.float64), group, 1)[:, :q.shape[1]]


def gelu(x):
    return 0.5 * x * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (x + 0.044715 * x ** 3)))


def matvec(x, w, bias=None, residual=None, act=False):
    """y in 64 bits and how far an fp32 result may be from it.

    An element of x is held to 2^-31 of the largest of its 128 (and to 2^-127), a rounding of half that; its
    products with levels and a group's sum are exact. Joining the digits' sums rounds five times, the scale's
    product and the groups' sums twice for each group, those of 16 warps and four digits once each: at most
    k / 16 + 27 times 2^-24 of the sum of magnitudes. Bias, GELU (of slope at most 1.13; tanhf and its products a few
    2^-24 of the value) and residual add a rounding each."""
    k = x.shape[1]
    wide = np.zeros((len(x), -(-k // 128) * 128))
    wide[:, :k] = np.abs(x)
    tops = np.repeat(wide.reshape(len(x), -1, 128).max(-1), 128, 1)[:, :k]
    held = (np.maximum(tops * 2.0 ** -31, 2.0 ** -127)) @ np.abs(w).T
    y = x.astype(np.float64) @ w.T
    err = (np.abs(x).astype(np.float64) @ np.abs(w).T) * (k / 16 + 27) * EPS + held
    if bias is not None:
        y = y + bias
        err = err + np.abs(y) * EPS
    if act:
        err = 1.13 * err + 12 * EPS * (np.abs(y) + 1e-30)
        y = gelu(y)
    if residual is not None:
        y = y + residual
        err = err + np.abs(y) * EPS
    return y, err


def rows_at(pages, scales, entries, n):
    """The first n positions [n, H, 64] (64 bits) of a sequence whose pages are `entries`, and which are mapped."""
    at = np.arange(n)
    e = np.asarray(entries)[at // PAGE] if n else np.zeros(0, np.int64)
    ok = (e >= 0) & (e < pages.shape[0])
    e0 = np.where(ok, e, 0)
    x = pages[e0, at % PAGE].astype(np.float64).reshape(n, -1, D)
    if scales is not None:
        x = x * scales[e0, :, at % PAGE].astype(np.float64)[..., None]
    return x, ok


def attention(q, k_pages, v_pages, table, row_start, ctx, heads, scale, out, max_new, k_scales=None, v_scales=None,
              prefix_table=None, prefix_lens=None, group_start=None):
    """`out` with the rows of the batch filled in (64 bits), and for each element the largest |v| that the row sees and
    the largest scale * sum |q||k| of its scores, which the error bound takes (ops_oracle.attention_bound)."""
    out = np.array(out, np.float64)
    vmax, smax = np.zeros(out.shape), np.zeros(out.shape)
    kv_heads = k_pages.shape[2] // D
    group = heads // kv_heads
    n_seq, width = table.shape
    for s in range(n_seq):
        lo, hi = int(row_start[s]), int(row_start[s + 1])
        if lo < 0 or hi <= lo or hi > len(q) or hi - lo > max_new or ctx[s] < 0 or ctx[s] + hi - lo > width * PAGE:
            continue
        n = int(ctx[s]) + hi - lo
        parts = []
        if prefix_table is not None:
            for g in range(len(prefix_lens)):
                a, b, m = int(group_start[g]), int(group_start[g + 1]), int(prefix_lens[g])
                if 0 <= a <= s < b <= n_seq and 0 < m <= prefix_table.shape[1] * PAGE:
                    parts.append((prefix_table[g], m, False))
        parts.append((table[s], n, True))
        ks, vs, ok, pos = [], [], [], []
        for entries, m, own in parts:
            k, good = rows_at(k_pages, k_scales, entries, m)
            v, _ = rows_at(v_pages, v_scales, entries, m)
            ks.append(k)
            vs.append(v)
            ok.append(good)
            pos.append(np.arange(m) if own else np.full(m, -1))
        k, v, ok, pos = (np.concatenate(x) for x in (ks, vs, ok, pos))
        for r in range(lo, hi):
            seen = ok & (pos <= ctx[s] + r - lo)
            kk, vv = k[seen], v[seen]
            for h in range(heads):
                c = slice(h * D, (h + 1) * D)
                if not len(kk):
                    out[r, c] = 0.0
                    continue
                x, y = kk[:, h // group], vv[:, h // group]
                with np.errstate(all="ignore"):
                    t = scale * (x @ q[r, c].astype(np.float64))
                    p = np.exp(t - t.max())
                    out[r, c] = (p / p.sum()) @ y
                    vmax[r, c] = np.abs(y).max()
                    smax[r, c] = abs(scale) * (np.abs(x) @ np.abs(q[r, c]).astype(np.float64)).max()
    return out, vmax, smax
