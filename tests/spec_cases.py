"""Plain 64-bit forms of the speculative-decoding operators (numpy), and random trees, for their tests."""
import numpy as np

U32 = 2.0 ** -24  # half a step of f32, relative
U16 = 2.0 ** -11  # half a step of f16


def random_tree(n, rng, back=8, unused=0, roots=0.0):
    """parent[n]: each node under one of the `back` before it (or a root), the last `unused` places empty."""
    parent = np.array([-1] + [-1 if rng.random() < roots else int(rng.integers(max(0, t - back), t)) for t in range(1, n)],
                      np.int32)
    parent[n - unused:] = -2
    return parent


def ancestors(parent):
    """[n][n] bool: which nodes each one sees; no row for an unused place."""
    n = len(parent)
    sees = np.zeros((n, n), bool)
    for t in range(n):
        if parent[t] < -1:
            continue
        u = t
        while True:
            sees[t, u] = True
            p = int(parent[u])
            if not 0 <= p < u or parent[p] < -1:
                break
            u = p
    return sees


def rope(x, pos, freq, mscale, n_rot, interleaved, norm=None, eps=0.0):
    """x [n][heads][hd] -> the turned heads, and a bound on an f32 computation's error (absolute, per element)."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    angle = pos.astype(np.float64)[:, None, None] * freq
    c, s = mscale * np.cos(angle), mscale * np.sin(angle)
    i = np.arange(n_rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n_rot // 2)
    y, size = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = mscale * (np.abs(x[..., a]) + np.abs(x[..., b]))
    # c and s rounded once, a product, the sum (and the norm's three: scale, product, weight): each half a step of size
    return y, size * U32 * (6.5 if norm is not None else 3.5)


def tree_attention(q, kc, vc, kd, vd, past, parent):
    """q [n][nh][hd], caches [nkv][..][hd], drafted rows [nkv][n][hd] -> out [n][nh][hd] and its bound per row."""
    n, nh, hd = q.shape
    rep = nh // kc.shape[0]
    sees = ancestors(parent)
    out, tol = np.zeros(q.shape), np.zeros((n, nh, 1))
    for t in range(n):
        if parent[t] < -1:
            continue
        for h in range(nh):
            g = h // rep
            k = np.concatenate([kc[g, :past], kd[g][sees[t]]]).astype(np.float64)
            v = np.concatenate([vc[g, :past], vd[g][sees[t]]]).astype(np.float64)
            qv = q[t, h].astype(np.float64)
            s = k @ qv / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ v
            # a score: hd products and sums in f32, in any order, its scaling and the exponent's argument (base 2); the
            # weights: their exponential and the sums over the positions, of which a fixed order adds parts of parts, and
            # the merge (2 * 64 additions at most count for a term)
            ds = (hd + 4) * U32 * (np.abs(k) @ np.abs(qv)).max() / np.sqrt(hd) + 4 * U32 * np.abs(s).max()
            tol[t, h] = (2 * ds + (128 + hd) * U32) * (p @ np.abs(v)).max() + 2 * ds * np.abs(out[t, h]).max()
    return out, tol


def sample(x, temp, top_k, top_p, min_p, u):
    """One row: the token and its probability among the kept."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if x.max() == -np.inf:
        return -1, 0.0
    best = int(np.argmax(x))
    if not temp > 0:
        return best, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == x[best], 1.0, np.where((x == -np.inf) | (x[best] == np.inf), 0.0,
                                                 np.exp((x - x[best]) / np.float64(temp))))
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        order = order[(before < np.float64(top_p) * w[order].sum()) | (np.arange(len(order)) == 0)]
    order = order[(w[order] >= np.float64(min_p)) | (np.arange(len(order)) == 0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    at = min(int((run <= np.float64(np.clip(u, 0, None)) * run[-1]).sum()), len(kept) - 1)
    while w[kept[at]] == 0:  # u at its upper end
        at -= 1
    return int(kept[at]), w[kept[at]] / run[-1]


def accepted(token, parent, sampled, room):
    """The accepted path."""
    if room <= 0 or parent[0] < -1:
        return []
    path = [0]
    while len(path) < room:
        nxt = [t for t in range(path[-1] + 1, len(token)) if parent[t] == path[-1] and token[t] == sampled[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    return path
