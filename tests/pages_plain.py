"""Plain statements of the operators over cache pages (ob_pages_*), in numpy: attention in float64, the choice of pages in the rounding that its
definition names, moves by indexing."""
import numpy as np

PAGE = 16


def bits16(shape, r, kind, std=1.0):
    """Random values of a 16-bit type as float64, and the same as the type's bits."""
    x = (r.standard_normal(shape) * std).astype(np.float32)
    return to16(x, kind)


def to16(x, kind):
    x = np.asarray(x, np.float32)
    if kind == "f16":
        h = x.astype(np.float16)
        return h.astype(np.float64), h.view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    b = ((u + 0x7fff + (u >> 16 & 1)) >> 16).astype(np.uint16)
    b[np.isnan(x)] = 0x7fc0
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64), b


def positions(pool, table, n, n_pages):
    """[n, kv, dim] of the first n positions of a sequence, and which of them are there."""
    out = np.zeros((n,) + (pool.shape[1], pool.shape[3]))
    there = np.zeros(n, bool)
    for x in range(n):
        if x // PAGE < len(table) and 0 <= table[x // PAGE] < n_pages:
            out[x], there[x] = pool[table[x // PAGE], :, x % PAGE], True
    return out, there


def attend(q, k, v, seen, scale):
    """q [heads, dim], k and v [n, kv, dim], seen [n]: output [heads, dim] and what its error scales with: the largest |v|, sum |q k| and count."""
    heads, kv = q.shape[0], k.shape[1]
    out = np.zeros((heads, v.shape[2]))
    size = np.zeros(heads), np.zeros(heads)
    k, v = k[seen], v[seen]
    if len(k):
        for h in range(heads):
            kh, vh = k[:, h * kv // heads], v[:, h * kv // heads]
            s = kh @ q[h] * scale
            w = np.exp(s - s.max())
            out[h] = (w / w.sum()) @ vh
            size[0][h], size[1][h] = np.abs(vh).max(), (np.abs(kh) @ np.abs(q[h])).max() * scale
    return out, size[0], size[1], len(k)


def tree(q, k, v, tables, first, n_ctx, visible, scale, out, tol_of):
    """Writes the tokens' outputs into `out` and the bounds of their errors into the array it returns."""
    tol = np.zeros(out.shape[:2])
    for s in range(len(n_ctx)):
        m = first[s + 1] - first[s]
        if m <= 0:
            continue
        n = n_ctx[s] + m
        ks, there = positions(k, tables[s], n, k.shape[0])
        vs, _ = positions(v, tables[s], n, k.shape[0])
        for t in range(m):
            seen = there.copy()
            for j in range(m):
                seen[n_ctx[s] + j] &= visible[first[s] + t] >> j & 1 == 1
            o, a, b, c = attend(q[first[s] + t], ks, vs, seen, scale)
            out[first[s] + t] = o
            tol[first[s] + t] = tol_of(a, b, c)
    return tol


def listed(q, k, v, tables, n_pos, selected, scale, row_seq, tol_of):
    """q [rows, heads, dim], selected [rows, kv, n]: outputs and the bounds of their errors."""
    rows, heads, dim = q.shape
    kv = k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros((rows, heads))
    for r in range(rows):
        s = row_seq[r]
        if not 0 <= s < len(tables):
            continue
        for g in range(kv):
            x = np.array([p * PAGE + i for p in selected[r, g] if 0 <= p < len(tables[s]) and 0 <= tables[s][p] < k.shape[0] for i in range(PAGE) if p * PAGE + i < n_pos[r]], int)
            page, slot = np.asarray(tables[s])[x // PAGE], x % PAGE
            hs = slice(g * heads // kv, (g + 1) * heads // kv)
            o, a, b, c = attend(q[r, hs], k[page, g, slot][:, None], v[page, g, slot][:, None], np.ones(len(x), bool), scale)
            out[r, hs], tol[r, hs] = o, tol_of(a, b, c)
    return out, tol


def bounds(k, tables, first_pos, n_pos, codes, scales):
    """Writes the touched pages' codes and units (float32 arithmetic, as defined)."""
    for s in range(len(n_pos)):
        for p in range(first_pos[s] // PAGE, -(-n_pos[s] // PAGE)):
            if first_pos[s] >= n_pos[s] or p >= len(tables[s]) or not 0 <= tables[s][p] < k.shape[0]:
                continue
            rows = k[tables[s][p], :, :min(PAGE, n_pos[s] - p * PAGE)].astype(np.float32)
            hi, lo = np.fmax.reduce(rows, 1), np.fmin.reduce(rows, 1)
            hi, lo = (np.clip(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf), np.float32(-1e18), np.float32(1e18)) for x in (hi, lo))
            d = np.maximum(np.abs(hi), np.abs(lo)).max(-1) / np.float32(127)
            by = np.where(d > 0, d, np.float32(1))[:, None]
            codes[tables[s][p], :, 0] = np.clip(np.ceil(hi / by), -127, 127)
            codes[tables[s][p], :, 1] = np.clip(np.floor(lo / by), -127, 127)
            scales[tables[s][p]] = d


def select(q, codes, scales, tables, n_pos, n, keep_first, keep_last, row_seq, kv):
    """[rows, kv, n] page numbers within the sequence, -1 behind the last."""
    rows, heads, dim = q.shape
    out = np.full((rows, kv, n), -1, np.int32)
    q = np.clip(np.nan_to_num(q.astype(np.float32), nan=0.0, posinf=np.inf, neginf=-np.inf), np.float32(-1e18), np.float32(1e18))
    for r in range(rows):
        s = row_seq[r]
        if not 0 <= s < len(tables):
            continue
        count = -(-int(n_pos[r]) // PAGE)
        table = np.asarray(tables[s][:count])
        there = (table >= 0) & (table < len(codes))
        for g in range(kv):
            best = np.full(count, -np.inf, np.float32)
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                d = np.abs(q[r, h]).max() / np.float32(127)
                c = np.clip(np.rint(q[r, h] / (d if d > 0 else np.float32(1))), -127, 127).astype(np.int64)
                b = codes[np.where(there, table, 0), g].astype(np.int64)
                whole = np.maximum(c * b[:, 0], c * b[:, 1]).sum(-1).astype(np.float32)
                best = np.maximum(best, d * scales[np.where(there, table, 0), g] * whole)
            rank = np.where(there, best.astype(np.float64), -np.inf)
            rank[:keep_first] = np.inf
            rank[max(0, count - keep_last):] = np.inf
            # keep_first + keep_last is at most n, so that all of those are taken; equals go by their number
            order = sorted(range(count), key=lambda p: (-rank[p], p))[:n]
            out[r, g, :len(order)] = sorted(order)
    return out
