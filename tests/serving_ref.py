"""Plain statements, in 64 bits, of the serving operators (numpy, one thing at a time)."""
import numpy as np

PAGE = 64


def rope(x, table, pos, rot, interleaved, inverse=False):
    """[rows, heads, hd] turned to positions `pos` by the table's entries."""
    y = np.array(x, dtype=np.float64)
    for j in range(rot // 2):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
        c, s = (np.asarray(table, dtype=np.float64)[pos, j, i][:, None] for i in (0, 1))
        s = -s if inverse else s
        va, vb = np.float64(1) * x[:, :, a], np.float64(1) * x[:, :, b]
        y[:, :, a], y[:, :, b] = va * c - vb * s, va * s + vb * c
    return y


def held(x, kind):
    """What the cache holds of f32 rows [..., hd]: each operation of the rounding in f32, as the library states it."""
    x = np.asarray(x, dtype=np.float32)
    f32 = np.float32
    with np.errstate(all="ignore"):
        if kind == "f16":
            y = np.clip(x, f32(-65504), f32(65504)).astype(np.float16).astype(np.float64)
            return np.where(np.isfinite(x), y, np.nan)
        b = x.reshape(*x.shape[:-1], -1, 32)
        if kind == "q8_0":
            d = np.minimum(np.abs(b).max(-1) * (f32(1) / f32(127)), f32(65504)).astype(np.float16)
        else:
            hi, lo = b.max(-1), b.min(-1)
            d = np.clip(np.where(hi > -lo, hi, lo) * f32(-0.125), f32(-65504), f32(65504)).astype(np.float16)
        f = d.astype(f32)
        inv = np.where(f != 0, f32(1) / np.where(f != 0, f, f32(1)), f32(0)).astype(f32)
        c = np.rint(b * inv[..., None])
        c = np.clip(c, -127, 127) if kind == "q8_0" else np.clip(c, -8, 7)
        y = c.astype(np.float64) * f.astype(np.float64)[..., None]
        y = np.where(np.isfinite(b).all(-1)[..., None], y, np.nan)
        return y.reshape(x.shape)


def attention(q, k, v, scale):
    """q [n_q, hd]; k, v [n_kv, n, hd] -> [n_q, hd]; no positions: zeros."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    if k.shape[1] == 0:
        return np.zeros_like(q)
    g = q.shape[0] // k.shape[0]
    out = np.empty_like(q)
    for h in range(q.shape[0]):
        s = k[h // g] @ q[h] * scale
        e = np.exp(s - s.max())
        out[h] = e @ v[h // g] / e.sum()
    return out


def penalised(l, penalty, recent):
    l = np.array(l, dtype=np.float32)
    for t in recent:
        if 0 <= t < len(l):
            l[t] = np.float32(l[t] / np.float32(penalty)) if l[t] > 0 else np.float32(l[t] * np.float32(penalty))
    return l


def kept(l, temperature, top_k, top_p, min_p):
    """(ids in order of logit, weights of all ids in 64 bits) of one row."""
    l = np.asarray(l, dtype=np.float64)
    fine = ~np.isnan(l) & (l > -np.inf)
    w = np.zeros(len(l))
    if not fine.any():
        return np.array([], dtype=int), w
    best = l[fine].max()
    if not temperature > 0:
        w[np.flatnonzero(fine & (l == best))[0]] = 1.0
        return np.flatnonzero(w), w
    with np.errstate(all="ignore"):
        w[fine] = np.where(l[fine] == best, 1.0, np.exp((l[fine] - best) / np.float64(temperature)))
    order = np.flatnonzero(fine)
    order = order[np.lexsort((order, -l[order]))]
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order]) - w[order]
        order = order[(mass < top_p * w[order].sum()) | (np.arange(len(order)) == 0)]
    return order[w[order] >= min(min_p, 1.0)], w


def sample(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability, how far the draw is from a border of its token, over the sum) of one row."""
    order, w = kept(l, temperature, top_k, top_p, min_p)
    ids = np.sort(order)
    if len(ids) == 0:
        return -1, 0.0, 1.0
    cum = np.cumsum(w[ids])
    i = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(ids) - 1)
    edges = np.abs(cum - u * cum[-1])[: len(ids) - 1]
    return int(ids[i]), w[ids[i]] / cum[-1], float(edges.min() / cum[-1]) if len(edges) else 1.0
