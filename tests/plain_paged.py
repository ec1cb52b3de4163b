"""The operators over a paged cache from their definitions, in 64 bits, position by position: what the kernels are held to.  Pages are arrays
[n_pages, page_size, n_head_kv, d] of float64, tables lists of page ids."""
import numpy as np

HALF_STEP = {"F16": 2.0 ** -11, "BF16": 2.0 ** -8, "F32": 2.0 ** -24}   # a rounding's largest error relative to the value
SMALLEST = {"F16": 2.0 ** -25, "BF16": 2.0 ** -134, "F32": 2.0 ** -150}  # half the distance of subnormal numbers


def rounded(x, ty):
    """the nearest value of the type (ties to even), as float64"""
    if ty == "F16":
        return np.asarray(x, dtype=np.float64).astype(np.float16).astype(np.float64)
    f = np.ascontiguousarray(x, dtype=np.float32)
    if ty == "F32":
        return f.astype(np.float64)
    u = f.view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)


def bits(x, ty):
    """values of the type as they lie in memory"""
    if ty == "F32":
        return np.ascontiguousarray(x, dtype=np.float32)
    if ty == "F16":
        return np.ascontiguousarray(x, dtype=np.float16).view(np.uint16)
    return (np.ascontiguousarray(x, dtype=np.float32).view(np.uint32) >> 16).astype(np.uint16)


def values(raw, ty):
    """the inverse, as float64"""
    if ty == "F32":
        return raw.view(np.float32).astype(np.float64)
    if ty == "F16":
        return raw.view(np.float16).astype(np.float64)
    return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rope_rows(n, d, n_dims, base=10000.0):
    """(cos, sin) rows by position, float32, pair i at 2 i and 2 i + 1"""
    angle = np.arange(n)[:, None] * base ** (-np.arange(0, n_dims, 2) / max(n_dims, 1))
    rows = np.zeros((n, d), dtype=np.float32)
    rows[:, 0:n_dims:2], rows[:, 1:n_dims:2] = np.cos(angle), np.sin(angle)
    return rows


def rotated(x, row, n_dims, mode):
    """x [heads, d] turned by one table row -> (values, sum of the two products' magnitudes)"""
    y, size = x.astype(np.float64).copy(), np.abs(x.astype(np.float64))
    for i in range(n_dims // 2):
        a, b = (2 * i, 2 * i + 1) if mode == 0 else (i, i + n_dims // 2)
        c, s = float(row[2 * i]), float(row[2 * i + 1])
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
        size[:, a] = size[:, b] = np.abs(x[:, a]) + np.abs(x[:, b])
    return y, size


def cell(tables, seq, pos, page_size, n_pages):
    """(page, place in it) of a position, None where table or page id do not reach"""
    if not 0 <= seq < len(tables) or pos < 0 or pos // page_size >= len(tables[seq]):
        return None
    page = tables[seq][pos // page_size]
    return (page, pos % page_size) if 0 <= page < n_pages else None


def append(k_pages, v_pages, tables, q, k, v, pos, seq, rows, n_dims, mode):
    """-> (q_out, k_pages, v_pages, the magnitudes for q_out and k_pages, tokens left out, tokens with an index out of range); unrounded; NaN in q_out: untouched"""
    ps, n_pages = k_pages.shape[1], k_pages.shape[0]
    kp, vp, qo = k_pages.copy(), v_pages.copy(), np.full(q.shape, np.nan)
    ks, qs = np.zeros(k_pages.shape), np.zeros(q.shape)
    bad = 0
    for t in range(len(pos)):
        if pos[t] < 0:
            continue
        at = cell(tables, int(seq[t]), int(pos[t]), ps, n_pages)
        if at is None or (n_dims and pos[t] >= len(rows)):
            bad += 1
            continue
        row = rows[pos[t]] if n_dims else None
        qo[t], qs[t] = rotated(q[t], row, n_dims, mode)
        kp[at], ks[at] = rotated(k[t], row, n_dims, mode)
        vp[at] = v[t]
    return qo, kp, vp, qs, ks, bad


def attention(k_pages, v_pages, tables, q, lens, shared, group_first, scale, sinks=None):
    """q [n_seq, heads, d] -> (out, sum of w |v|, largest |v| seen, sum of exp(score - largest))"""
    n_seq, heads, d = q.shape
    ps, n_pages, kv = k_pages.shape[1], k_pages.shape[0], k_pages.shape[2]
    out, size, big, total = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n_seq, heads, 1)), np.ones((n_seq, heads, 1))
    first_of = list(range(n_seq))
    for g in range(len(group_first) - 1):
        for s in range(group_first[g], group_first[g + 1]):
            first_of[s] = group_first[g]
    for s in range(n_seq):
        at = [cell(tables, first_of[s] if p < shared[s] else s, p, ps, n_pages) for p in range(lens[s])]
        at = [x for x in at if x is not None]
        if not at:
            continue
        page, place = np.array(at).T
        for h in range(heads):
            kk, vv = k_pages[page, place, h * kv // heads], v_pages[page, place, h * kv // heads]
            x = kk @ q[s, h] * scale
            top = x.max() if sinks is None else max(x.max(), float(sinks[h]))
            if top == -np.inf:
                continue
            w = np.exp(x - top)
            z = w.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - top))
            seen = w > 0
            out[s, h], size[s, h] = w[seen] @ vv[seen] / z, w[seen] @ np.abs(vv[seen]) / z
            # of the finite ones: a channel that holds another has no bound of this kind, and bounds no other channel
            big[s, h], total[s, h] = np.abs(np.where(np.isfinite(vv[seen]), vv[seen], 0.0)).max(initial=0.0), z
    return out, size, big, total


def select(logits, scores, k, done=None, end_token=0):
    """logits [requests, beams, vocab] -> (scores, tokens, parents), each [requests, k]"""
    R, B, V = logits.shape
    out = np.full((R, k), -np.inf), np.full((R, k), -1, dtype=np.int64), np.full((R, k), -1, dtype=np.int64)
    for r in range(R):
        found = []
        for b in range(B):
            if not scores[r, b] > -np.inf:
                continue
            if done is not None and done[r, b]:
                found.append((-float(scores[r, b]), b, end_token))
                continue
            x = np.where(np.isnan(logits[r, b]), -np.inf, logits[r, b].astype(np.float64))
            top = x.max()
            if top == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                off = np.where(x == top, 0.0, x - top)
            gain = float(scores[r, b]) + (off - np.log(np.exp(off).sum()))
            best = np.lexsort((np.arange(V), -gain))[:k]
            found += [(-gain[w], b, int(w)) for w in best if gain[w] > -np.inf]
        for i, (s, b, w) in enumerate(sorted(found)[:k]):
            out[0][r, i], out[1][r, i], out[2][r, i] = -s, w, b
    return out


def reorder(parents, tables, lens, page_size, pools):
    """parents [requests, beams]; tables, lens by sequence; pools: arrays [n_pages, ...] -> (tables, lens, row_of, pools)"""
    R, B = len(parents), len(parents[0])
    pools = [p.copy() for p in pools]
    new_tables, new_lens, row_of = [], [], []
    for r in range(R):
        par = [p if 0 <= p < B else -1 for p in parents[r]]
        free = [b for b in range(B) if b not in par]
        row = [None] * B
        for j, p in enumerate(par):
            if p >= 0 and p not in par[:j]:
                row[j] = p
        for j, p in enumerate(par):
            if p >= 0 and row[j] is None:
                row[j] = free.pop(0)
                n = lens[r * B + p]
                for i, (f, t) in enumerate(zip(tables[r * B + p], tables[r * B + row[j]])):
                    if i * page_size < n and f != t:
                        for pool in pools:
                            if 0 <= f < len(pool) and 0 <= t < len(pool):
                                pool[t] = pool[f]
        for j, p in enumerate(par):
            if row[j] is None:
                row[j] = free.pop(0)
            row_of.append(row[j])
            new_tables.append(list(tables[r * B + row[j]]))
            new_lens.append(lens[r * B + p] if p >= 0 else 0)
    return new_tables, new_lens, row_of, pools
