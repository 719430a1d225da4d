"""Plain statements, in numpy and 64 bits, of 4-bit pages, of the attention of new tokens with weights added up, of cutting caches down, and of the
verification of drafted tokens."""
import numpy as np

PAGE, GROUP, LARGEST = 16, 32, 7168.0


def in_four_bits(x):
    """What entries x [..., dim] stand for once they are kept in 4 bits: an exponent and a ceiling at a time."""
    x = np.asarray(x, np.float64)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -LARGEST, LARGEST).reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = x.max(-1), x.min(-1)
    a = np.maximum(hi, -lo) / 8
    step = np.ldexp(1.0, np.maximum(np.frexp(a)[1] - 7, -24))  # a is from 64 to 128 of them
    d = np.where(hi > -lo, -1.0, 1.0) * np.ceil(a / step) * step
    c = np.clip(np.rint(x / np.where(d != 0, d, 1.0)[..., None]), -8, 7)
    return (c * d[..., None]).reshape(*x.shape[:-2], -1)


def seen_by(first, n_ctx, visible, s, n_positions):
    """Which positions token t of sequence s sees: [tokens, positions]."""
    m = int(first[s + 1] - first[s])
    x = np.arange(n_positions)
    if visible is None:
        return x[None] <= n_ctx[s] + np.arange(m)[:, None]
    out = np.zeros((m, n_positions), bool)
    for t in range(m):
        j = x - n_ctx[s]
        out[t] = (j < 0) | np.array([0 <= v < 64 and visible[first[s] + t] >> int(v) & 1 == 1 for v in j])
    return out


def attend_tokens(q, k, v, there, first, n_ctx, visible, scale, out, mass, rel_of, rounded=0.0):
    """q [tokens, heads, dim]; k, v: per sequence [positions, kv, dim]; there: per sequence which positions exist.  Writes out and mass [sequences, kv, positions];
    returns the bounds of their errors.  rel_of(qk, n): a weight's relative error where sum |q k| is at most qk and n positions are seen;
    rounded: that of the weights on their way into the products with values, which goes into sum w v as it is."""
    tol, mass_tol = np.zeros(out.shape[:2]), None if mass is None else np.zeros(mass.shape)
    kv = k[0].shape[1] if len(k) else 1
    group = q.shape[1] // kv
    for s in range(len(n_ctx)):
        m = int(first[s + 1] - first[s])
        if m <= 0:
            continue
        n = min(int(n_ctx[s]) + m, len(k[s]))
        sees = seen_by(first, n_ctx, visible, s, n) & there[s][None, :n]
        for h in range(kv):
            kh, vh = np.where(there[s][:n, None], k[s][:n, h], 0.0), np.where(there[s][:n, None], v[s][:n, h], 0.0)
            got, got_tol = np.zeros(n), np.zeros(n)
            for t in range(m):
                for g in range(group):
                    x = q[first[s] + t, h * group + g]
                    e, size = kh @ x * scale, (np.abs(kh) @ np.abs(x)).max(initial=0.0) * scale
                    if not sees[t].any():
                        out[first[s] + t, h * group + g] = 0.0
                        continue
                    w = np.where(sees[t], np.exp(np.where(sees[t], e - e[sees[t]].max(), 0.0)), 0.0)
                    w /= w.sum()
                    out[first[s] + t, h * group + g] = w @ vh
                    rel = rel_of(size, n)
                    tol[first[s] + t, h * group + g] = (2 * rel + rounded) * (w @ np.abs(vh)).max() + np.abs(vh[sees[t]]).max() * (n * 2.0 ** -32 + 2.0 ** -22)
                    got += w
                    got_tol += 2 * rel * w + 2.0 ** -40
            if mass is not None:
                c = min(int(n_ctx[s]), n)
                row, row_tol = mass[s, h], mass_tol[s, h]
                old = np.where(np.arange(n) < c, row[:n], 0.0)
                row[:n] = np.where(there[s][:n], old + got, row[:n])
                # rounded at each of the rows' sums (m group of them) and once when added
                row_tol[:n] = np.where(there[s][:n], got_tol + (m * group + 4) * 2.0 ** -24 * got + 2.0 ** -23 * np.abs(row[:n]), 0.0)
    return tol, mass_tol


def evict(mass, n_pos, n_keep, keep_first, keep_last):
    """kept [layers, sequences, kv, n_keep] and the lengths afterwards."""
    layers, seqs, kv, _ = mass.shape
    kept = np.full((layers, seqs, kv, n_keep), -1, np.int32)
    for s in range(seqs):
        n = int(n_pos[s])
        for li in range(layers):
            for h in range(kv):
                if n <= n_keep:
                    kept[li, s, h, :n] = np.arange(n)
                    continue
                rank = [(np.inf if i < keep_first or i >= n - keep_last else -np.inf if np.isnan(mass[li, s, h, i]) else float(mass[li, s, h, i])) for i in range(n)]
                level = [1 if i < keep_first or i >= n - keep_last else 0 for i in range(n)]
                nan = [0 if np.isnan(mass[li, s, h, i]) and not level[i] else 1 for i in range(n)]
                order = sorted(range(n), key=lambda i: (-level[i], -nan[i], -rank[i], i))[:n_keep]
                kept[li, s, h] = sorted(order)
    return kept, np.minimum(n_pos, n_keep).astype(np.int32)


def verify(target, draft, tokens, parent, first, uniform, width=64):
    """The rule as it is stated for distributions: the residual is normalised after each rejection."""
    clean = lambda x: np.where((x > 0) & np.isfinite(x), x, 0.0).astype(np.float64)  # noqa: E731
    n = len(first) - 1
    kept, count, token = np.full((n, width), -1, np.int32), np.zeros(n, np.int32), np.full(n, -1, np.int32)
    vocab = target.shape[1]
    for s in range(n):
        a, nodes = int(first[s]), min(64, int(first[s + 1] - first[s]))
        if nodes <= 0:
            continue
        at, path = 0, [0]
        while True:
            p = clean(target[a + at])
            r, went, total = p.copy(), False, 1.0
            q = None if draft is None else clean(draft[a + at])
            for j in range(at + 1, nodes):
                x = int(tokens[a + j])
                if parent[a + j] != at or not 0 <= x < vocab:
                    continue
                u = max(0.0, float(uniform[a + j]))
                if u * (total if q is None else q[x]) < r[x]:
                    at, went = j, True
                    path.append(j)
                    break
                if q is None:
                    total, r[x] = max(0.0, total - r[x]), 0.0
                elif r.any():
                    r = np.maximum(r - q, 0.0)
                    r = r / r.sum() if r.sum() > 0 else r
            if not went:
                break
        if not r.sum() > 0:
            r = p
        upto = np.cumsum(r)
        if upto[-1] > 0:
            token[s] = min(int(np.searchsorted(upto, max(0.0, float(uniform[a])) * upto[-1], side="right")), int(np.flatnonzero(r)[-1]))
        count[s] = min(len(path), width)
        kept[s, :count[s]] = path[:width]
    return kept, count, token
