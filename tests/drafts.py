"""The operators of sampled and speculated decoding in 64 bits, from their
definitions."""
import numpy as np

NONE = 0xFFFFFFFF


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability, kept words) of one row of logits."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore"):
        words = np.flatnonzero(x > -np.inf)
    if words.size == 0:
        return NONE, 0.0, words
    order = words[np.argsort(-(x[words] + np.float32(0)), kind="stable")]
    if temperature == 0:
        order = order[:1]
    elif top_k:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        d = np.where(x[order] == top, 0.0, x[order].astype(np.float64) - np.float64(top))
        w = np.where(d == 0.0, 1.0, np.exp(d / np.float64(np.float32(temperature))) if temperature else 0.0)
    c = np.cumsum(w)
    n = len(w)
    if top_p < 1.0:
        n = int(np.argmax(c >= np.float64(np.float32(top_p)) * c[-1])) + 1
    n = max(1, min(n, int((w >= np.float64(np.float32(min_p))).sum())))
    at = np.argsort(order[:n])
    kept, w = order[:n][at], w[:n][at]
    c = np.cumsum(w)
    u = float(np.float32(u)) if u > 0 else 0.0
    j = int(np.searchsorted(c, u * c[-1], side="right"))
    j = min(j, int(np.flatnonzero(w).max()))
    return int(kept[j]), w[j] / c[-1], kept


def random_tree(rng, n, bushy=1.5):
    return [-1] + [int(i * rng.random() ** bushy) for i in range(1, n)]


def ancestors(parents):
    a = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            a[i] = a[p]
        a[i, i] = True
    return a


def mask_words(seen):
    n = seen.shape[0]
    w = (n + 31) // 32
    b = np.zeros((n, 32 * w), np.uint64)
    b[:, :n] = seen
    return (b.reshape(n, w, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)


def rotate(x, pos, freq, rope_dim, halves, scale=1.0, f32_angle=False):
    """x [n, heads, head_dim] f64 rotated at positions pos"""
    th = np.outer(np.asarray(pos, np.float64), np.asarray(freq[:rope_dim // 2], np.float64))
    if f32_angle:
        th = th.astype(np.float32).astype(np.float64)
    i = np.arange(rope_dim // 2)
    a, b = (i, i + rope_dim // 2) if halves else (2 * i, 2 * i + 1)
    y = np.array(x, np.float64)
    c, s = scale * np.cos(th)[:, None], scale * np.sin(th)[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def attend(q, k, v, seen, scale):
    """q [n, n_head, hd], k, v [n_kv, P, hd], seen [n, P] -> (out [n, n_head, hd]
    in f64, how far f32-grade arithmetic may be from it, by element's row)

    A score: q kept to 2^-22 of the row's largest element, its hd products
    added in f32 (each partial sum's rounding below 2^-24 of the sum of
    magnitudes, hd + 2 of them in the worst order); a probability: the score's
    error relative, 2^-22 of hi + lo and 2^-22 of exp2; the sums over P
    positions and their split, 2^-24 per step of the at most 64 + P / 32 steps
    that follow one another, all of it against the largest |v|."""
    n, H, D = q.shape
    g = H // k.shape[0]
    out, tol = np.zeros(q.shape), np.zeros((n, H, 1))
    k, v = k.astype(np.float64), v.astype(np.float64)
    for h in range(H):
        with np.errstate(invalid="ignore"):
            s = q[:, h].astype(np.float64) @ k[h // g].T * scale
        s = np.where(seen, s, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0.0)), 0.0)
        l = p.sum(1, keepdims=True)
        p = p / np.where(l > 0, l, 1.0)
        for i in range(n):
            out[i, h] = p[i][seen[i]] @ v[h // g][seen[i]]
        mag = np.where(seen, np.abs(q[:, h]).astype(np.float64) @ np.abs(k[h // g]).T, 0.0).max(1)
        big = np.where(seen, np.abs(q[:, h]).max(1, keepdims=True) * np.abs(k[h // g]).sum(1)[None], 0.0).max(1)
        ds = scale * (2.0 ** -22 * big + (D + 2) * 2.0 ** -24 * mag) + 2.0 ** -22 * (1 + np.abs(np.where(np.isfinite(m[:, 0]), m[:, 0], 0)))
        vmax = np.abs(np.where(np.isfinite(v[h // g]), v[h // g], 0)).max()
        tol[:, h, 0] = vmax * (2 * ds + 2.0 ** -21 + (64 + k.shape[1] / 32) * 2.0 ** -24)
    return out, tol
