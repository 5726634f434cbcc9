"""A paged cache in 64 bits, by plain loops over sequences and heads: what tests/test_gpu_paged.py grades against.
Works on the CPU from copies of the device's tensors."""
import numpy as np

EPS = 2.0 ** -24  # half a step of f32, relative


def places(table, b, n, page):
    """Pool row of sequence b's rows 0..n-1."""
    s = np.arange(n)
    return table[b][s // page].astype(np.int64) * page + s % page


def rotate(x, pos, theta):
    """x [n, heads, d] turned to positions pos .. pos + n - 1, column i paired with column i + d / 2."""
    half = x.shape[-1] // 2
    ang = (pos + np.arange(len(x), dtype=np.float64))[:, None] / theta ** (2 * np.arange(half) / x.shape[-1])
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    lo, hi = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate((lo * c - hi * s, hi * c + lo * s), -1)


def attend(q, k, v, table, q_start, n_rows, page, H, Hkv, d):
    """(out, lse, weights [B, Hkv, max rows], bound): q [N, H, d], k/v [pool rows, Hkv, d].

    bound [N, H, d] is how far f32 arithmetic may take out.  A score is a sum of d products, each rounded, scaled and
    stored: it is off by at most (d + 4) EPS sum |q k| / sqrt d =: e, so that a weight is off by a factor within e^(+-2 e) of
    its exact value (its own score and the normaliser's), and the exponential and the division add a few EPS; sums over n keys
    add n EPS of the sum of absolute terms, rescaling once per tile of 16 keys another EPS each."""
    g = H // Hkv
    out = np.zeros(q.shape)
    lse = np.zeros(q.shape[:2])
    bound = np.zeros(q.shape)
    w = np.zeros((len(n_rows), Hkv, max(max(n_rows), 1)))
    w_bound = np.zeros_like(w)
    for b, n in enumerate(n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        at = places(table, b, n, page)
        for h in range(H):
            kk, vv = k[at, h // g].astype(np.float64), v[at, h // g].astype(np.float64)
            for t in range(t0, t1):
                m = n - (t1 - t) + 1
                qt = q[t, h].astype(np.float64)
                s = kk[:m] @ qt / np.sqrt(d)
                lse[t, h] = s.max() + np.log(np.exp(s - s.max()).sum())
                p = np.exp(s - lse[t, h])
                out[t, h] = p @ vv[:m]
                e = 2 * (d + 4) * EPS * (np.abs(kk[:m]) @ np.abs(qt)).max() / np.sqrt(d)
                rel = np.expm1(e) + (m + m / 16 + 32) * EPS
                bound[t, h] = rel * (p @ np.abs(vv[:m]))
                w[b, h // g, :m] += p
                w_bound[b, h // g, :m] += rel * p
            w_bound[b, h // g] += g * (t1 - t0) * EPS * w[b, h // g]
    return out, lse, w, bound, w_bound


def evict(w, n, budget, first, last):
    """The rows that one head keeps."""
    rows = np.arange(n)
    if n <= budget:
        return rows
    middle = rows[first:n - last]
    nan = np.isnan(w[middle])
    x = np.where(nan, np.float32(-np.inf), w[middle]).astype(np.float64)
    best = middle[np.lexsort((middle, nan, -x))[:budget - first - last]]
    return np.sort(np.concatenate((rows[:first], best, rows[n - last:])))


def rows_kind(rows, d):
    """The launch kind of so many rows per kv head (new tokens x heads of the group): their limit, 0 for the last kind."""
    dp = 32 * -(-d // 32)
    kinds = [16, 32, 64, 128] if dp <= 128 else [16, 64] if dp <= 192 else [16]
    return next((k for k in kinds if rows <= k), 0)


# (heads, kv heads, width) for batch_of_kinds; the same with the most rows per kv head for batch_of_few.
KIND_SHAPES = [(8, 8, 32), (16, 8, 50), (8, 8, 64), (24, 8, 96), (32, 8, 128), (16, 8, 192), (16, 8, 256)]
FEW_SHAPES = [(8, 8, 32, 16), (8, 8, 32, 32), (16, 8, 64, 16), (16, 8, 64, 32), (16, 8, 50, 32), (24, 8, 96, 16),
              (32, 8, 128, 16), (32, 8, 128, 32), (16, 8, 192, 16), (32, 8, 256, 16)]


def batch_of_kinds(H, Hkv):
    """(rows, new tokens) of 74 sequences that need every kind at once, each with too many workgroups or steps to join
    another's launch: 70 with one token, among them four with 24, 60, 120 and 400 rows per kv head."""
    g = H // Hkv
    ones = [(400 + (i * 37) % 500, 1) for i in range(70)]
    longs = [(7300, 120 // g), (900, 400 // g), (7300, 24 // g), (7300, 60 // g)]
    return list(zip(*(ones[:30] + longs[:2] + ones[30:] + longs[2:])))


def batch_of_few(H, Hkv, rows):
    """(rows, new tokens) of sequences with at most `rows` rows per kv head, 16 or 32, all of one launch kind."""
    most = rows // (H // Hkv)
    return [5000, 2700, 900, 65, 1300], [most, most - 1, most, most - 2, max(most - 3, rows // 2 // (H // Hkv) + 1)]
