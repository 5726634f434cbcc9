"""Trees of new tokens, rotary positions and shared pages in 64 bits, by plain loops: what tests/test_gpu_tree.py grades
against.  Works on the CPU from copies of the device's tensors."""
import numpy as np

from pagedref import EPS, places


def random_tree(rng, n, wide=1.5):
    """Parents of n tokens, wide near the first for a large exponent; -1 for the first and a few others."""
    up = np.floor(rng.random(n) ** wide * np.arange(n)).astype(np.int32)
    up[rng.random(n) < 0.05] = -1
    if n:
        up[0] = -1
    return up


def lines(parent):
    """Each token's own number and its ancestors'; a parent that is not an earlier token is none."""
    got = []
    for i, p in enumerate(parent):
        got.append((got[p] if 0 <= p < i else []) + [i])
    return got


def masks(parents, words):
    """uint64 [tokens, words] of a list of trees, and each token's depth."""
    N = sum(map(len, parents))
    got, depth, t0 = np.zeros((N, words), np.uint64), np.zeros(N, np.int32), 0
    for parent in parents:
        for i, p in enumerate(parent):
            if 0 <= p < i:
                got[t0 + i], depth[t0 + i] = got[t0 + p], depth[t0 + p] + 1
            got[t0 + i, i // 64] |= np.uint64(1 << (i % 64))
        t0 += len(parent)
    return got, depth


def seen(mask, n, L):
    """bool [L, n]: which of a sequence's n rows each of its L new tokens sees; mask [L, words]."""
    s = np.zeros((L, n), bool)
    s[:, :n - L] = True
    for t in range(L):
        for j in range(t + 1):
            s[t, n - L + j] = bool(int(mask[t, j // 64]) >> (j % 64) & 1)
    return s


def attend(q, k, v, table, q_start, n_rows, page, H, Hkv, d, sees):
    """(out, lse, bound): q [N, H, d], k/v [pool rows, Hkv, d], sees: seen(...) of each sequence.  The bound is
    pagedref.attend's, for the rows that a token sees."""
    g = H // Hkv
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    for b, n in enumerate(n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        at = places(table, b, n, page)
        for h in range(H):
            kk, vv = k[at, h // g].astype(np.float64), v[at, h // g].astype(np.float64)
            for t in range(t0, t1):
                own = sees[b][t - t0]
                m = int(own.sum())
                if m == 0:
                    continue
                qt = q[t, h].astype(np.float64)
                s = kk[own] @ qt / np.sqrt(d)
                lse[t, h] = s.max() + np.log(np.exp(s - s.max()).sum())
                p = np.exp(s - lse[t, h])
                out[t, h] = p @ vv[own]
                e = 2 * (d + 4) * EPS * (np.abs(kk[own]) @ np.abs(qt)).max() / np.sqrt(d)
                bound[t, h] = (np.expm1(e) + (n + n / 16 + 32) * EPS) * (p @ np.abs(vv[own]))
    return out, lse, bound


def frequencies(rot, theta, scaling="plain", factor=1.0, low=1.0, high=4.0, context=8192.0):
    got = []
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling == "base":
            f = (theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot)
        if scaling == "turns":
            r = context * f / (2 * np.pi)
            s = 0.0 if r <= low else 1.0 if r >= high else (r - low) / (high - low)
            f = (1 - s) * f / factor + s * f
        got.append(f)
    return np.array(got)


def turn(x, pos, freq, rot, inter, amplitude=1.0, back=False):
    """(y, bound): x [rows, heads, d].  The angle pos f is rounded once, and a cosine's error is at most its
    argument's and a step of its own: |angle| + 2 steps of 64 bits on each product's factor; then one rounding to f32."""
    y = x.astype(np.float64)
    bound = np.zeros(y.shape)
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        ang = pos.astype(np.float64) * freq[i]
        c, s = amplitude * np.cos(ang)[:, None], amplitude * (-1 if back else 1) * np.sin(ang)[:, None]
        lo, hi = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        y[..., a], y[..., b] = lo * c - hi * s, hi * c + lo * s
        off = 4 * (np.abs(ang)[:, None] + 4) * 2.0 ** -53 * abs(amplitude) * (np.abs(lo) + np.abs(hi))
        bound[..., a] = bound[..., b] = off
    return y, bound + EPS * np.abs(y)


class Pages:
    """Tables and counts, changed as the entry points say."""

    def __init__(self, table, refs, page):
        self.table, self.refs, self.page = table.copy(), refs.copy(), page

    def pages(self, rows):
        return -(-rows // self.page)

    def fork(self, src, dst, n_rows, n_room):
        """(pairs, missing)."""
        before, pairs, takes = self.refs.copy(), np.full((len(src), 2), -1, np.int32), []
        for i, (a, b, n, room) in enumerate(zip(src, dst, n_rows, n_room)):
            for j in range(n // self.page, self.pages(room)):
                p = self.table[a, j]
                if a != b or not (0 <= p < len(before) and before[p] == 1):
                    takes.append((i, j))
        free = np.nonzero(before == 0)[0]
        if len(takes) > len(free):
            return pairs, len(takes) - len(free)
        old = self.table.copy()
        for a, b, n in zip(src, dst, n_rows):
            if a == b:
                continue
            self.table[b] = -1
            for j in range(n // self.page):
                p = self.table[b, j] = old[a, j]
                if 0 <= p < len(before):
                    self.refs[p] += 1
        for (i, j), f in zip(takes, free):
            a, b, n = src[i], dst[i], n_rows[i]
            p = old[a, j]
            self.table[b, j] = f
            self.refs[f] += 1
            if a == b and 0 <= p < len(before):
                self.refs[p] -= 1
            if j == n // self.page and n % self.page:
                pairs[i] = p, f
        return pairs, 0

    def free(self, n_keep):
        for b, n in enumerate(n_keep):
            for j in range(min(self.pages(n), self.table.shape[1]), self.table.shape[1]):
                p = self.table[b, j]
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
                self.table[b, j] = -1

    def compact(self, most):
        """(pairs, moved)."""
        live = np.nonzero(self.refs)[0]
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        high = [p for p in live[::-1] if p >= len(live)]
        assert len(holes) == len(high)
        pairs, now = np.full((most, 2), -1, np.int32), np.arange(len(self.refs), dtype=np.int32)
        for i, (to, of) in enumerate(list(zip(holes, high))[:most]):
            pairs[i] = of, to
            now[of] = to
            self.refs[to], self.refs[of] = self.refs[of], 0
        named = (self.table >= 0) & (self.table < len(now))
        self.table = np.where(named, now[np.where(named, self.table, 0)], self.table).astype(np.int32)
        return pairs, [min(most, len(holes)), max(0, len(holes) - most)]

    def counted(self):
        """References by the table."""
        named = self.table[(self.table >= 0) & (self.table < len(self.refs))]
        return np.bincount(named, minlength=len(self.refs))
