"""Plain 64-bit implementations of attention over a paged cache, and of what
cache_assign and cache_compact do to tables and pages (numpy and Python lists,
on the host), with the bound that the attention's arithmetic keeps.  It counts
roundings of u = 2^-24 (half a step of fp32, relative)."""
import numpy as np

from operators_ref import U, half_step


def keys_of(cache, table, n, page):
    """Tokens 0 .. n - 1 of one head: (values [n, dim], which are there) of cache [pages, page, dim] (float64)."""
    out, there = np.zeros((n, cache.shape[-1])), np.zeros(n, bool)
    for e in range(min(len(table), -(-n // page))):
        if 0 <= table[e] < len(cache):
            got = cache[table[e]][:n - e * page]
            out[e * page:e * page + len(got)], there[e * page:e * page + len(got)] = got, True
    return out, there


def attention(q, k_cache, v_cache, tables, positions, counts, scale=None, softcap=0.0, window=0, slopes=None, slots=None, f16=False):
    """(out, bound) of q [rows, heads, dim] over caches [pages, heads, page, dim].

    Scores: a product of dim terms (dim roundings at most, and two of 2^-22 of
    fp32 q's two parts, of the sum of the absolute products), the cap (its function
    good to 2^-21 of the cap's value), the bias (two roundings of it) and the
    exponent (three of the score).  An error of dx in every score changes a weight's
    share by 2 dx.  Weights enter the products as fp16 (2^-11; fp32 q: two parts,
    2^-21); sums over n keys take a rounding per 16 keys and one for every part and
    rescaling: (n / 8 + 64) u of the sum of absolute terms."""
    q, kc, vc = (np.asarray(t, np.float64) for t in (q, k_cache, v_cache))
    rows, heads, dim = q.shape
    page, group = kc.shape[2], heads // kc.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, bound = np.zeros_like(q), np.zeros_like(q)
    start = 0
    for s, n in enumerate(counts):
        slot = s if slots is None else slots[s]
        table = tables[slot] if 0 <= slot < len(tables) else []
        most = max(0, min(positions[s] + n, len(table) * page))
        for j in range(kc.shape[1]):
            k, there = keys_of(kc[:, j], table, most, page)
            v, _ = keys_of(vc[:, j], table, most, page)
            for h in range(j * group, (j + 1) * group):
                for t in range(n):
                    p, r = positions[s] + t, start + t
                    lo = max(0, p + 1 - window) if window else 0
                    see = np.flatnonzero(there[lo:max(lo, min(p + 1, most))]) + lo
                    if not len(see):
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = scale * (k[see] @ q[r, h])
                        size = abs(scale) * (np.abs(k[see]) @ np.abs(q[r, h]))
                        dx = size.max() * ((dim + 8) * U + 2.0 ** -21) + 4 * U * np.abs(x).max()
                        if softcap:
                            x = softcap * np.tanh(x / softcap)
                            dx += softcap * 2.0 ** -21
                        if slopes is not None:
                            x = x + slopes[h] * (see - p)
                            dx += 3 * U * np.abs(slopes[h] * (see - p)).max()
                        dx += 4 * U * min(np.ptp(x), 40.0)
                        w = np.exp(x - x.max())
                        w /= w.sum()
                        out[r, h] = w @ v[see]
                        bound[r, h] = (2 * dx + (2.0 ** -11 if f16 else 2.0 ** -20) + (len(see) / 8 + 64) * U) * (w @ np.abs(v[see])) + half_step(
                            out[r, h], f16) + 1e-30
        start += n
    return out, bound


def assign(pages, page, tables, lengths, parents, counts):
    """(new tables, new lengths, missing, copies (from, to, tokens))."""
    slots, width = len(tables), len(tables[0]) if tables else 0
    length = [min(max(lengths[p], 0), width * page) if 0 <= p < slots else 0 for p in parents]

    def there(p):
        return p if 0 <= p < pages else -1
    full = [[there(tables[p][e]) for e in range(n // page)] if n else [] for p, n in zip(parents, length)]
    held = {p for t in full for p in t if p >= 0}
    shared, new, jobs = set(held), [list(t) for t in full], []
    for s, (p, n) in enumerate(zip(parents, length)):
        if n % page:
            last = there(tables[p][n // page])
            if last < 0:
                new[s].append(-1)
            elif last in shared:
                jobs.append((s, last, n % page))
            else:
                shared.add(last)
                new[s].append(last)
    free, missing = [p for p in range(pages) if p not in shared], 0
    for s in range(slots):
        need = -(-(length[s] + max(0, counts[s])) // page)
        for e in range(len(new[s]), need):
            if e >= width or not free:
                missing += 1
            if e < width:
                new[s].append(free.pop(0) if free else -1)
    copies = [(p, new[s][length[s] // page], n) for s, p, n in jobs if new[s][length[s] // page] >= 0]
    return [t + [-1] * (width - len(t)) for t in new], length, missing, copies


def compact(pages, page, tables, lengths):
    """(new tables, pages held, moves (from, to))."""
    width = len(tables[0]) if tables else 0
    held = [[p if e * page < min(n, width * page) and 0 <= p < pages else -1 for e, p in enumerate(t)] for t, n in zip(tables, lengths)]
    used = sorted({p for t in held for p in t if p >= 0})
    n = len(used)
    moves = dict(zip([p for p in used if p >= n], sorted(set(range(n)) - set(used))))
    return [[moves.get(p, p) for p in t] for t in held], n, list(moves.items())
