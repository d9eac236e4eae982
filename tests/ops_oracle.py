"""64-bit definitions of the operators over the paged cache, for the tests (numpy, CPU)."""
import numpy as np

PAGE, D = 16, 64
OK, CAPACITY, ARG, DEVICE = 0, 8, 10, 11


def pages_of(n):
    return (n + PAGE - 1) // PAGE


def plan(ctx, new, table, n_pages, max_rows, free=None, n_free=0):
    """(table, n_free, row_start, seq_of, pos_of, slot_of, status)"""
    table = np.array(table)
    n, width = table.shape
    seq, pos, slot = (np.full(max_rows, -1, np.int64) for _ in range(3))
    start = np.zeros(n + 1, np.int64)

    def refused(status):
        return table, n_free, start, seq, pos, slot, status

    if min(ctx) < 0 or min(new) < 0 or (free is not None and not 0 <= n_free <= len(free)):
        return refused(ARG)
    need = sum(pages_of(c + m) - pages_of(c) for c, m in zip(ctx, new)) if free is not None else 0
    if max(c + m for c, m in zip(ctx, new)) > width * PAGE or sum(new) > max_rows or need > n_free:
        return refused(CAPACITY)
    out = table.copy()
    r = 0
    for s, (c, m) in enumerate(zip(ctx, new)):
        if free is not None:
            for j in range(pages_of(c), pages_of(c + m)):
                n_free -= 1
                out[s, j] = free[n_free]
        for p in range(c, c + m):
            e = out[s, p // PAGE]
            seq[r], pos[r] = s, p
            slot[r] = e * PAGE + p % PAGE if 0 <= e < n_pages else -1
            r += 1
        start[s + 1] = r
    return out, n_free, start, seq, pos, slot, OK


def attention(q, k_pages, v_pages, table, row_start, ctx, heads, kv_heads, scale, out):
    """Fills the rows of `out` (float64 copy of what was there) and returns it with each row's
    error unit: the largest |v| it sees and the largest scale * sum |q||k| of its scores."""
    out = np.array(out, np.float64)
    vmax, smax = np.zeros(out.shape), np.zeros(out.shape)
    n_pages = k_pages.shape[0]
    group = heads // kv_heads
    for s in range(len(ctx)):
        lo, hi = row_start[s], row_start[s + 1]
        for r in range(lo, hi):
            n = ctx[s] + r - lo + 1
            e = table[s, np.arange(n) // PAGE]
            seen = (e >= 0) & (e < n_pages)
            e, row = e[seen], (np.arange(n) % PAGE)[seen]
            for h in range(heads):
                c = slice(h * D, (h + 1) * D)
                if not len(e):
                    out[r, c] = 0.0
                    continue
                g = slice(h // group * D, (h // group + 1) * D)
                k, v = k_pages[e, row, g], v_pages[e, row, g]
                t = scale * (k @ q[r, c])
                p = np.exp(t - t.max())
                out[r, c] = (p / p.sum()) @ v
                vmax[r, c] = np.abs(v).max()
                smax[r, c] = abs(scale) * (np.abs(k) @ np.abs(q[r, c])).max()
    return out, vmax, smax


def attention_bound(vmax, smax, length):
    """How far an fp32 result may be from the exact one.

    A score is a sum of 64 products: in fp32, or as hi . hi + hi . lo + lo . hi of operands split into two
    16-bit terms of 11 significant bits each (what is dropped or rounded of a product is at most 3 x 2^-22 of
    it), its relative error against sum |q||k| is at most (64 + 12 + 4) 2^-24, in units of the score after
    scaling. exp turns an error e of the score into a factor exp(e); 2^x adds 2^-22, the running rescale and
    the sums of `length` terms at most (length + 64) 2^-24, the product with v its split again (12 x 2^-24).
    Numerator and denominator both carry the error, hence twice."""
    eps = 2.0 ** -24
    return vmax * 2.0 * (np.expm1(80 * eps * smax) + (length + 96) * eps)


def beam_select(logits, scores, done, beams, eos):
    """(next, parent, scores, done) by place, from the definition."""
    n, vocab = logits.shape
    nxt, par, sc, dn = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros(n), np.zeros(n, np.int64)
    for q in range(n // beams):
        cand = []
        for b in range(beams):
            i = q * beams + b
            if done is not None and done[i]:
                cand.append((scores[i] if scores[i] == scores[i] else -np.inf, b * vocab + eos))
                continue
            x = np.where(np.isnan(logits[i]), -np.inf, logits[i]).astype(np.float64)
            m = x.max()
            with np.errstate(all="ignore"):
                t = scores[i].astype(np.float64) + (x - (m + np.log(np.exp(x - m).sum()))) if np.isfinite(m) \
                    else np.full(vocab, -np.inf)
            t = np.where(np.isnan(t), -np.inf, t)
            best = np.lexsort((np.arange(vocab), -t))[:beams]
            cand += [(t[v], b * vocab + v) for v in best]
        cand.sort(key=lambda c: (-c[0], c[1]))
        kept = cand[:beams]
        place, taken = {}, set()
        for c in kept:
            b = c[1] // vocab
            if b not in taken:
                taken.add(b)
                place[c] = b
        free = iter(sorted(set(range(beams)) - taken))
        for c in kept:
            p = q * beams + (place[c] if c in place else next(free))
            b, v = divmod(c[1], vocab)
            nxt[p], par[p], sc[p] = v, q * beams + b, c[0]
            dn[p] = int(bool(done is not None and done[q * beams + b]) or v == eos)
    return nxt, par, sc, dn


def reorder(pages, table, parent, first, length, beams):
    """pages [layers, n_pages, 16, w] after the reorder."""
    new, n_pages = pages.copy(), pages.shape[1]
    for s, p in enumerate(parent):
        r = s // beams
        if p == s or p // beams != r or p < 0:
            continue
        for pos in range(max(first[r], 0), min(length[r], table.shape[1] * PAGE)):
            a, b = table[p, pos // PAGE], table[s, pos // PAGE]
            if a != b and 0 <= a < n_pages and 0 <= b < n_pages:
                new[:, b, pos % PAGE] = pages[:, a, pos % PAGE]
    return new
