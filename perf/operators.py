"""The paged KV cache's operators, as cases that can be timed and checked: the append of new tokens, the attention of
a chunk of new tokens (one token and more) with or without the accumulation of its weights, and the eviction that
keeps the rows with the largest accumulated weight.

A sequence's row s lies in row s % page_size of the page that its page table names at s / page_size; pages are
[page_size, Hkv * d], f32.  The batch is ragged: new tokens are packed one sequence after the other, and each
sequence's new tokens are its cache's last rows.  With `own` false the operators are computed in their plain form
(gathers into a padded batch, products, exp, sums), else by the C ABI of libzt_attn.so on the caller's buffers.
"""
import importlib.util
import math
import os

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA = 500000.0

# (query heads, kv heads, head width): those of the contiguous caches' cases.
HEADS = [(4, 2, 32), (8, 8, 64), (32, 8, 128), (32, 8, 96), (16, 4, 256), (12, 4, 64)]
MAX_BYTES = 64 * 8192 * 8 * 128 * 4  # K of the largest cache below
MAX_PAIRS = 32 * 128 * 2048 * 4096   # H d x visible pairs of the largest prompt below


def listed():
    return [
        # One token of the small model goes into its cache: a launch and its host side.
        dict(name="append_one", kind="append", B=1, rows=129, spread=0, chunk=1, every=1, few=1, page=16, H=4, Hkv=2, d=32),
        # Prompts of different lengths go into their pages, behind a part that is there already.
        dict(name="append_prompts", kind="append", B=7, rows=1003, spread=611, chunk=512, every=1, few=1, page=64, H=32, Hkv=8, d=128),
        # One sequence answers, token by token, on a long cache: latency.
        dict(name="decode_one", kind="attend", B=1, rows=4096, spread=0, chunk=1, every=1, few=1, page=16, H=32, Hkv=8, d=128),
        # Serving: 64 sequences of different lengths, a token each.
        dict(name="decode_batch", kind="attend", B=64, rows=8192, spread=4096, chunk=1, every=1, few=1, page=64, H=32, Hkv=8, d=128),
        # Four drafted tokens of each sequence are checked at once; a group of three heads, small pages.
        dict(name="draft_four", kind="attend", B=16, rows=2047, spread=1201, chunk=4, every=1, few=4, page=8, H=12, Hkv=4, d=64),
        # A chunk of one prompt against a partly filled cache.
        dict(name="chunk_one", kind="attend", B=1, rows=2340, spread=0, chunk=333, every=1, few=1, page=16, H=32, Hkv=8, d=128),
        # Prompts' chunks among sequences that answer: every fourth brings 501 tokens, the others one.
        dict(name="mixed_batch", kind="attend", B=12, rows=3001, spread=1500, chunk=501, every=4, few=1, page=32, H=32, Hkv=8, d=96),
        # A whole long prompt.
        dict(name="prompt", kind="attend", B=1, rows=4096, spread=0, chunk=4096, every=1, few=1, page=64, H=32, Hkv=8, d=128),
        # Tokens whose attention weights are accumulated for the eviction.
        dict(name="weights_decode", kind="weights", B=16, rows=4096, spread=2048, chunk=1, every=1, few=1, page=16, H=32, Hkv=8, d=128),
        # The same for a prompt.
        dict(name="weights_prompt", kind="weights", B=1, rows=2048, spread=0, chunk=2048, every=1, few=1, page=64, H=32, Hkv=8, d=128),
        # A small cache gives up its lightest rows.
        dict(name="evict_small", kind="evict", B=1, rows=320, spread=0, page=16, budget=256, first=4, last=64, H=4, Hkv=2, d=32),
        # Full caches are cut to half, sequences below the budget among them.
        dict(name="evict_batch", kind="evict", B=16, rows=8192, spread=5000, page=64, budget=4096, first=4, last=512, H=32, Hkv=8, d=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "weights", "weights", "evict"])
    H, Hkv, d = rng.choice(HEADS)
    page = rng.choice([1, 8, 16, 16, 32, 64, 256])
    B = _log_int(rng, 1, 64)
    rows = _log_int(rng, 1, 8192)
    while B * rows * Hkv * d * 4 > MAX_BYTES // (1 if kind == "attend" else 4):
        B = (B + 1) // 2
        rows = rows * 3 // 4
    case = dict(kind=kind, B=B, rows=rows, spread=rng.randrange(0, rows), page=page, H=H, Hkv=Hkv, d=d)
    if kind == "evict":
        budget = rng.randrange(1, rows + 1)
        first = min(budget, rng.choice([0, 1, 4, 16]))
        case.update(budget=budget, first=first, last=rng.randrange(0, budget - first + 1))
        return case
    chunk = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 2, 16), _log_int(rng, 17, max(17, rows)),
                        _log_int(rng, 17, max(17, rows))])
    while chunk > 1 and B * H * d * chunk * rows > MAX_PAIRS:
        chunk = chunk * 3 // 4
    case.update(chunk=chunk, every=rng.choice([1, 1, 2, 4]), few=rng.choice([0, 1, 1, 3]))
    return case


def _lengths(case):
    """(rows of each sequence after the append, new tokens of each): the same for every seed."""
    rows, spread = case["rows"], case["spread"]
    n = [rows - (spread * ((i * 37) % 64 + 1) // 64 if spread else 0) for i in range(case["B"])]
    if case["kind"] == "evict":
        return n, [0] * len(n)
    return n, [min(r, case["chunk"] if i % case["every"] == 0 else case["few"]) for i, r in enumerate(n)]


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


def _inputs(case, seed):
    """The case's tensors, from the seed alone, and the host's arrays."""
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 12345)
    B, page, H, Hkv, d = case["B"], case["page"], case["H"], case["Hkv"], case["d"]
    n_rows, q_len = _lengths(case)
    evict = case["kind"] == "evict"

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    used = [(n + page - 1) // page for n in n_rows]
    out_used = [(min(n, case["budget"]) + page - 1) // page for n in n_rows] if evict else []
    stride = max(used)
    n_pages = sum(used) + sum(out_used) + 2  # some pages are nobody's
    pages = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)
    x = dict(n_rows=np.array(n_rows, dtype=np.int32), q_start=np.cumsum([0] + q_len, dtype=np.int32), n_pages=n_pages,
             w_stride=max(n_rows))

    def table(counts, at):  # a sequence's pages, and behind them entries that name no page
        t = torch.full((B, stride), -1, device="cuda", dtype=torch.int32)
        for b, c in enumerate(counts):
            t[b, :c] = pages[at:at + c]
            at += c
        return t

    x["table"] = table(used, 0)
    x["k"], x["v"] = normal(n_pages, page, Hkv * d), normal(n_pages, page, Hkv * d)
    N = int(x["q_start"][-1])
    if evict:
        # Accumulated weights are sums of probabilities: many small, few large; rows of the same weight among them.
        w = torch.rand(B, Hkv, max(n_rows), device="cuda", generator=gen) ** 4 * 8
        x["w"] = torch.where(w < 0.25, torch.floor(w * 256) / 256, w)
        x["table_out"] = table(out_used, sum(used))
        x["w_out"] = torch.zeros_like(x["w"])
        x["kept"] = torch.empty(B, Hkv, case["budget"], device="cuda", dtype=torch.int32)
        return x
    x["q"] = normal(N, H * d)
    if case["kind"] == "append":
        x["k_new"], x["v_new"] = normal(N, Hkv * d), normal(N, Hkv * d)
        x["q_out"] = torch.empty_like(x["q"])
        x["w_out"] = torch.rand(B, Hkv, max(n_rows), device="cuda", generator=gen)
        # Positions run on after an eviction: they are past the rows.
        x["pos"] = np.array([n - q + 1000 * (i % 3) for i, (n, q) in enumerate(zip(n_rows, q_len))], dtype=np.int32)
        return x
    x["out"] = torch.empty_like(x["q"])
    x["lse"] = torch.empty(N, H, device="cuda")
    if case["kind"] == "weights":
        x["w"] = torch.rand(B, Hkv, max(n_rows), device="cuda", generator=gen)
        x["w_out"] = torch.zeros_like(x["w"])
    return x


def prepare(case, seed):
    return dict(case=case, ws=None, **_inputs(case, seed))


def _pool_rows(s, table, n):
    """Row of the pool for each sequence's row 0..n-1 (rows past its last: row 0 of the pool)."""
    page = s["case"]["page"]
    at = torch.arange(n, device="cuda")
    rows = table[:, at // page].long() * page + at % page
    return rows.clamp_(min=0), at


def _padded(s):
    """(token of each sequence's padded slot, whether the slot is one, rows of each sequence, row of each slot)."""
    q_start = torch.from_numpy(s["q_start"]).cuda().long()
    n_rows = torch.from_numpy(s["n_rows"]).cuda().long()
    q_len = q_start[1:] - q_start[:-1]
    i = torch.arange(max(1, int((s["q_start"][1:] - s["q_start"][:-1]).max())), device="cuda")
    is_token = i[None, :] < q_len[:, None]
    token = torch.where(is_token, q_start[:-1, None] + i[None, :], 0)
    return token, is_token, n_rows, (n_rows - q_len)[:, None] + i[None, :]


def _rotated(x, heads, d, pos):
    """x [N, heads * d] turned to its rows' positions; angles, and the turn itself, in 64 bits."""
    half = d // 2
    angle = pos.double()[:, None] / THETA ** (torch.arange(half, device="cuda", dtype=torch.float64) / half)[None, :]
    c, sn = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    y = x.view(-1, heads, d).double()
    lo, hi = y[..., :half], y[..., half:]
    return torch.cat((lo * c - hi * sn, hi * c + lo * sn), -1).float().view(-1, heads * d)


def _plain_append(s):
    case = s["case"]
    H, Hkv, d, page = case["H"], case["Hkv"], case["d"], case["page"]
    _, is_token, _, row = _padded(s)
    pos0 = torch.from_numpy(s["pos"]).cuda().long()
    first = row[:, :1]
    pos = (pos0[:, None] + row - first)[is_token]
    b = torch.arange(case["B"], device="cuda")[:, None].expand_as(row)[is_token]
    row = row[is_token]
    at = s["table"][b, row // page].long() * page + row % page
    s["k"].view(-1, Hkv * d)[at] = _rotated(s["k_new"], Hkv, d, pos)
    s["v"].view(-1, Hkv * d)[at] = s["v_new"]
    s["w_out"].transpose(1, 2)[b, row] = 0.0
    return dict(q=_rotated(s["q"], H, d, pos), k=s["k"], v=s["v"], w=s["w_out"])


def _plain_attend(s):
    case = s["case"]
    B, H, Hkv, d = case["B"], case["H"], case["Hkv"], case["d"]
    g = H // Hkv
    token, is_token, n_rows, row = _padded(s)
    T, S = token.shape[1], int(s["n_rows"].max())
    rows, at = _pool_rows(s, s["table"], S)
    k = s["k"].view(-1, Hkv, d)[rows].permute(0, 2, 3, 1).contiguous().view(B * Hkv, d, S)
    v = s["v"].view(-1, Hkv, d)[rows].permute(0, 2, 1, 3).contiguous().view(B * Hkv, S, d)
    q = s["q"].view(-1, Hkv, g, d)[token].permute(0, 2, 3, 1, 4).contiguous().view(B * Hkv, g * T, d)
    score = torch.matmul(q, k).view(B, Hkv, g, T, S).mul_(_scale(case))
    hidden = (at[None, None, :] > row[:, :, None]) | (at[None, None, :] >= n_rows[:, None, None])
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total)
    o = torch.matmul(p.view(B * Hkv, g * T, S), v).view(B, Hkv, g, T, d)
    out = o.permute(0, 3, 1, 2, 4)[is_token].reshape(-1, H * d)
    lse = (top + total.log()).view(B, H, T).permute(0, 2, 1)[is_token]
    if case["kind"] == "attend":
        return dict(out=out, lse=lse)
    p.masked_fill_(~is_token[:, None, None, :, None], 0.0)
    mine = (at[None, :] < n_rows[:, None])[:, None, :]
    w = torch.where(mine, s["w"] + p.sum((2, 3)), s["w_out"])
    return dict(out=out, lse=lse, w=w)


def _plain_evict(s):
    case = s["case"]
    B, Hkv, d, page, budget = case["B"], case["Hkv"], case["d"], case["page"], case["budget"]
    n = torch.from_numpy(s["n_rows"]).cuda().long()[:, None, None]
    S = int(s["n_rows"].max())
    at = torch.arange(S, device="cuda")[None, None, :]
    # Kept in any case, in the choice, behind the last row.
    always = (at < case["first"]) | (at >= n - case["last"]) | (n <= budget)
    rank = torch.where(at >= n, 2, torch.where(always, 0, 1)).expand(B, Hkv, S)
    by_weight = s["w"].sort(dim=-1, descending=True, stable=True).indices
    by_rank = rank.gather(-1, by_weight).sort(dim=-1, stable=True).indices
    order = by_weight.gather(-1, by_rank)[..., :budget]
    order = torch.where(order < n, order, S).sort(dim=-1).values
    there = order < S
    kept = torch.where(there, order, -1).int()
    src, _ = _pool_rows(s, s["table"], S)
    dst, _ = _pool_rows(s, s["table_out"], order.shape[-1])
    b, h, j = torch.nonzero(there, as_tuple=True)
    r = order[b, h, j]
    k, v = s["k"].view(-1, Hkv, d), s["v"].view(-1, Hkv, d)
    k[dst[b, j], h] = k[src[b, r], h]
    v[dst[b, j], h] = v[src[b, r], h]
    s["w_out"][b, h, j] = s["w"][b, h, r]
    return dict(k=s["k"], v=s["v"], w=s["w_out"], kept=torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=-1))


_zt = None


def _lib():
    global _zt
    if _zt is None:
        path = os.path.join(ROOT, "z-transformer_amd", "zt_attn.py")
        spec = importlib.util.spec_from_file_location("zt_attn", path)
        _zt = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_zt)
    return _zt.lib()


def _done(rc):
    if rc != 0:
        raise RuntimeError("the library refused a call")


def _own_run(s):
    L, case = _lib(), s["case"]
    kind, B, page, H, Hkv, d = case["kind"], case["B"], case["page"], case["H"], case["Hkv"], case["d"]
    stream = torch.cuda.current_stream().cuda_stream
    n_rows, q_start = s["n_rows"].ctypes.data, s["q_start"].ctypes.data
    pool = (B, s["n_pages"], page, s["table"].shape[1], s["w_stride"])
    k, v, table = s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr()
    if kind == "append":
        _done(L.zt_paged_append(s["q"].data_ptr(), s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["q_out"].data_ptr(),
                                k, v, table, s["w_out"].data_ptr(), q_start, n_rows, s["pos"].ctypes.data, *pool, H, Hkv,
                                d, THETA, stream))
        return dict(q=s["q_out"], k=s["k"], v=s["v"], w=s["w_out"])
    if kind == "evict":
        _done(L.zt_paged_evict(k, v, table, s["table_out"].data_ptr(), s["w"].data_ptr(), s["w_out"].data_ptr(),
                               s["kept"].data_ptr(), n_rows, *pool, Hkv, d, case["first"], case["last"], case["budget"],
                               stream))
        return dict(k=s["k"], v=s["v"], w=s["w_out"], kept=s["kept"])
    weights = kind == "weights"
    if s["ws"] is None:  # a serving program keeps one
        nbytes = L.zt_attn_paged_workspace(q_start, n_rows, B, H, Hkv, d, int(weights))
        s["ws"] = torch.empty(max(nbytes, 16), device="cuda", dtype=torch.uint8)
    w_in, w_out = (s["w"].data_ptr(), s["w_out"].data_ptr()) if weights else (None, None)
    _done(L.zt_attn_paged(s["q"].data_ptr(), k, v, table, s["out"].data_ptr(), s["lse"].data_ptr(), w_in, w_out,
                          q_start, n_rows, *pool, H, Hkv, d, s["ws"].data_ptr(), s["ws"].numel(), stream))
    got = dict(out=s["out"], lse=s["lse"])
    if weights:
        got["w"] = s["w_out"]
    return got


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    return _plain_append(state) if kind == "append" else _plain_evict(state) if kind == "evict" else _plain_attend(state)


def work(case):
    H, Hkv, d = case["H"], case["Hkv"], case["d"]
    n_rows, q_len = _lengths(case)
    N = sum(q_len)
    if case["kind"] == "append":
        # q, k, v in; q out, k, v into the cache, a weight cleared.
        return dict(bytes=4 * (N * (2 * H + 4 * Hkv) * d + N * Hkv), flops=3 * N * (H + Hkv) * d)
    if case["kind"] == "evict":
        kept = sum(min(n, case["budget"]) for n in n_rows)
        # The weights read; each kept row's K and V read and written, its weight and its number written.
        return dict(bytes=4 * Hkv * (sum(n_rows) + kept * (4 * d + 2)), flops=0)
    seen = sum(n for n, q in zip(n_rows, q_len) if q)
    pairs = sum(q * n - q * (q - 1) // 2 for n, q in zip(n_rows, q_len))
    # q in, out and the log-sum-exp out, the K and V rows; the weights in and out.
    nbytes = 4 * (2 * N * H * d + N * H + 2 * seen * Hkv * d)
    if case["kind"] == "weights":
        nbytes += 8 * sum(n_rows) * Hkv
    return dict(bytes=nbytes, flops=4 * H * d * pairs)


def exact(case, seed):
    x = _inputs(case, seed)
    kind, B, page, H, Hkv, d = case["kind"], case["B"], case["page"], case["H"], case["Hkv"], case["d"]
    n_rows, q_start = x["n_rows"].tolist(), x["q_start"].tolist()

    def places(table, b, n):
        r = np.arange(n)
        t = table[b].cpu().numpy().astype(np.int64)
        return torch.from_numpy(t[r // page] * page + r % page).cuda()

    k, v = x["k"].view(-1, Hkv, d), x["v"].view(-1, Hkv, d)
    if kind == "evict":
        k, v, w_out, wn = k.double(), v.double(), x["w_out"].double(), x["w"].cpu().numpy()
        budget, first, last = case["budget"], case["first"], case["last"]
        kept = np.full((B, Hkv, budget), -1, np.int32)
        for b, n in enumerate(n_rows):
            src, dst = places(x["table"], b, n), places(x["table_out"], b, min(n, budget))
            for h in range(Hkv):
                rows = np.arange(n)
                if n > budget:
                    middle = rows[first:n - last]
                    best = middle[np.lexsort((middle, -wn[b, h, middle]))[:budget - first - last]]
                    rows = np.sort(np.concatenate((rows[:first], best, rows[n - last:])))
                kept[b, h, :len(rows)] = rows
                r = torch.from_numpy(rows).cuda()
                k[dst, h], v[dst, h] = k[src[r], h], v[src[r], h]
                w_out[b, h, :len(rows)] = x["w"][b, h, r].double()
        return dict(k=k.view_as(x["k"]), v=v.view_as(x["v"]), w=w_out, kept=torch.from_numpy(kept).cuda())
    if kind == "append":
        k, v, w = k.double(), v.double(), x["w_out"].double()

        def turned(rows, heads, pos):
            z = torch.view_as_complex(rows.double().view(-1, heads, 2, d // 2).transpose(2, 3).contiguous())
            angle = torch.arange(pos, pos + len(z), device="cuda", dtype=torch.float64)[:, None, None] * torch.pow(
                torch.tensor(THETA, device="cuda", dtype=torch.float64),
                -2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
            z = z * torch.polar(torch.ones_like(angle), angle)
            return torch.view_as_real(z).transpose(2, 3).reshape(-1, heads, d)

        q = torch.empty(q_start[-1], H, d, device="cuda", dtype=torch.float64)
        for b, n in enumerate(n_rows):
            t0, t1 = q_start[b], q_start[b + 1]
            if t1 > t0:
                at = places(x["table"], b, n)[n - (t1 - t0):]
                q[t0:t1] = turned(x["q"][t0:t1], H, int(x["pos"][b]))
                k[at] = turned(x["k_new"][t0:t1], Hkv, int(x["pos"][b]))
                v[at] = x["v_new"][t0:t1].view(-1, Hkv, d).double()
                w[b, :, n - (t1 - t0):n] = 0.0
        return dict(q=q.view(-1, H * d), k=k.view_as(x["k"]), v=v.view_as(x["v"]), w=w)
    g = H // Hkv
    out = torch.empty(q_start[-1], H, d, device="cuda", dtype=torch.float64)
    lse = torch.empty(q_start[-1], H, device="cuda", dtype=torch.float64)
    w = x["w_out"].double() if kind == "weights" else None
    q = x["q"].view(-1, H, d)
    for b, n in enumerate(n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        at = places(x["table"], b, n)
        for j in range(Hkv):
            if w is not None:
                w[b, j, :n] = x["w"][b, j, :n].double()
            if t1 == t0:
                continue
            kk, vv = k[at, j].double(), v[at, j].double()
            seen = torch.ones(t1 - t0, n, device="cuda", dtype=torch.bool).tril(n - (t1 - t0))
            for h in range(j * g, (j + 1) * g):
                score = (q[t0:t1, h].double() @ kk.t().contiguous()) / math.sqrt(d)
                score = torch.where(seen, score, -math.inf)
                lse[t0:t1, h] = torch.logsumexp(score, 1)
                p = torch.softmax(score, 1)
                out[t0:t1, h] = p @ vv
                if w is not None:
                    w[b, j, :n] += p.sum(0)
    got = dict(out=out.view(-1, H * d), lse=lse)
    if w is not None:
        got["w"] = w
    return got
