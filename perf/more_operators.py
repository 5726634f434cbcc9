"""The paged KV cache's operators for drafted trees and shared pages, as cases that can be timed and checked: rotary
positions of any layout, part and scale (a packed batch of q and k rows there and back, and the append of a tree's tokens to
the cache), the attention of a tree of drafted tokens, the move of the accepted ones' rows, and the forking, freeing,
compacting and copying of pages.

The cache is that of operators.py: a sequence's row s lies in row s % page_size of the page that its page table names
at s / page_size; pages are [page_size, Hkv * d], f32.  A sequence's new tokens are its cache's last rows.  They form a
tree: parent[i] is the number of token i's parent among them, an earlier one, or -1 where it follows the cache's
row before them; a token sees that row and all before it, its ancestors and itself.  A page is free
when nobody refers to it: refs counts the entries of page tables, here and elsewhere, that name it.  With `own` false the
operators are computed in their plain form, else by the C ABI of libzt_attn.so on the caller's buffers.
"""
import importlib.util
import math
import os

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA = 500000.0
# How the angles are scaled for contexts longer than the trained one: factor, and the turns within that context below
# which a frequency is divided by it and above which it is left alone.
FACTOR, LOW, HIGH, CONTEXT, AMPLITUDE = 8.0, 1.0, 4.0, 8192.0, 1.2079441541679836
SCALES = ["none", "linear", "base", "turns"]

# (query heads, kv heads, head width).
HEADS = [(4, 2, 32), (8, 8, 64), (32, 8, 128), (24, 8, 96), (16, 4, 256), (12, 4, 64)]
MAX_POOL = 24 * 5700 * 8 * 128         # values of K of the largest cache below
MAX_PAIRS = 32 * 128 * 24 * 41 * 5700  # H d x visible pairs of the largest trees below
MAX_ROWS = 40 * 128 * 8192             # values of the largest batch that is turned


def listed():
    return [
        # A tree of drafted tokens after one long sequence: latency.
        dict(name="tree_one", kind="tree", B=1, rows=4103, spread=0, nodes=26, page=16, H=32, Hkv=8, d=128),
        # Serving: the trees of 24 sequences of different lengths.
        dict(name="tree_batch", kind="tree", B=24, rows=8192, spread=5000, nodes=61, page=64, H=32, Hkv=8, d=128),
        # A few packed rows; neighbouring columns are pairs, three quarters of a head are turned.
        dict(name="turn_few", kind="turn", rows=37, far=4096, back=False, H=12, Hkv=4, d=64, rot=48, inter=True, scale="linear"),
        # The gradients of a training batch go back; positions scaled for a long context.
        dict(name="turn_back", kind="turn", rows=8192, far=65536, back=True, H=32, Hkv=8, d=128, rot=128, inter=False, scale="turns"),
        # A tree's tokens go into one cache.
        dict(name="append_one", kind="append", B=1, rows=1003, spread=0, nodes=26, page=16, H=32, Hkv=8, d=128, rot=128, inter=False, scale="turns"),
        # The trees of many sequences; half of a head is turned.
        dict(name="append_batch", kind="append", B=48, rows=2047, spread=1201, nodes=61, page=16, H=16, Hkv=4, d=256, rot=128, inter=True, scale="base"),
        # One tree's accepted tokens become its sequence's rows.
        dict(name="keep_one", kind="keep", B=1, rows=1003, spread=0, nodes=26, page=16, Hkv=8, d=128),
        # The same for many sequences.
        dict(name="keep_batch", kind="keep", B=64, rows=2047, spread=1201, nodes=61, page=16, Hkv=8, d=128),
        # Four beams of one sequence, in a pool that others use: the last step's are freed, this step's begin.
        dict(name="fork_few", kind="fork", B=2, rows=333, spread=0, beams=4, room=1, page=16, taken=211, spare=97, Hkv=2, d=32),
        # A batch's beams, and every fourth sequence is given room.
        dict(name="fork_batch", kind="fork", B=24, rows=4103, spread=3001, beams=4, room=64, page=64, taken=2003, spare=1009, Hkv=8, d=128),
        # A small pool gives its end back.
        dict(name="compact_small", kind="compact", B=3, rows=500, spread=100, moves=17, spare=40, page=16, Hkv=2, d=32),
        # A quarter of a large pool's pages move.
        dict(name="compact_large", kind="compact", B=24, rows=8192, spread=5000, moves=600, spare=1300, page=64, Hkv=8, d=128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "turn", "turn", "append", "keep", "fork", "fork", "compact"])
    H, Hkv, d = rng.choice(HEADS)
    turned = dict(H=H, Hkv=Hkv, d=d, rot=rng.choice([d, d, d // 2, d // 4 * 3, 2 * rng.randrange(2, d // 2 + 1)]),
                  inter=rng.choice([True, False]), scale=rng.choice(SCALES))
    if kind == "turn":
        rows = _log_int(rng, 1, MAX_ROWS // ((H + Hkv) * d))
        return dict(kind=kind, rows=rows, far=_log_int(rng, 16, 1 << 20), back=rng.choice([True, False]), **turned)
    page = rng.choice([1, 8, 16, 16, 32, 64, 256])
    B, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
    while B * rows * Hkv * d > MAX_POOL // (1 if kind in ("tree", "compact") else 3):
        B, rows = (B + 1) // 2, rows * 3 // 4 + 1
    while B * rows // page > 40000:
        page *= 2
    case = dict(kind=kind, B=B, rows=rows, spread=rng.randrange(0, rows), page=page)
    if kind in ("tree", "append", "keep"):
        nodes = rng.choice([1, _log_int(rng, 2, 16), _log_int(rng, 17, 80), _log_int(rng, 17, 80), _log_int(rng, 65, 600)])
        while nodes > 1 and B * H * d * nodes * rows > MAX_PAIRS:
            nodes = nodes * 3 // 4
        case.update(nodes=min(rows, nodes), **(turned if kind == "append" else dict(Hkv=Hkv, d=d)))
        if kind == "tree":
            case.update(H=H)
        return case
    case.update(Hkv=Hkv, d=d)
    pages = B * (rows // page + 1)
    if kind == "fork":
        case.update(beams=rng.choice([1, 2, 4, 8]), room=rng.choice([0, 1, page, _log_int(rng, 1, 300)]),
                    taken=rng.randrange(0, pages // 2 + 2), spare=rng.randrange(0, pages // 4 + 2))
        # A page that is somebody's is a page of the pool.
        while _fork_pages(case) * page * Hkv * d > MAX_POOL:
            case.update(beams=max(1, case["beams"] // 2), taken=case["taken"] // 2, spare=case["spare"] // 2, B=(case["B"] + 1) // 2,
                        room=case["room"] // 2)
        return case
    used = sum(-(-n // page) for n in _lengths(case))
    spare = rng.randrange(1, max(2, used // 3))
    case.update(spare=spare, moves=rng.randrange(0, min(spare, used) + 1))
    return case


def _lengths(case):
    """Rows of each sequence, the same for every seed."""
    rows, spread = case["rows"], case["spread"]
    return [rows - (spread * ((i * 37) % 64 + 1) // 64 if spread else 0) for i in range(case["B"])]


def _nodes(case):
    """New tokens of each sequence: all, two thirds, or a third of the most."""
    return [min(n, max(1, case["nodes"] * (3 - i % 3) // 3)) for i, n in enumerate(_lengths(case))]


def _fork_pages(case):
    n, page = _lengths(case), case["page"]
    used, want = [-(-x // page) for x in n], [-(-(x + case["room"]) // page) for x in n]
    fresh = [w - u if i % 4 == 3 else case["beams"] * (w - x // page) for i, (x, u, w) in enumerate(zip(n, used, want))]
    return sum(used) + sum(fresh) + case["taken"] + case["spare"]


def prepare(case, seed):
    """The case's tensors, from the seed alone, and the host's arrays."""
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 4242)
    rng = np.random.default_rng([seed, 77])
    kind, Hkv, d = case["kind"], case["Hkv"], case["d"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def ints(x):
        return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()

    s = dict(case=case, ws=None, freq=None)
    if kind == "turn":
        rows, H = case["rows"], case["H"]
        # Packed sequences of different lengths, each from a position of its own up.
        start = rng.integers(0, case["far"], size=rows // 100 + 1)
        at = np.arange(rows)
        s.update(pos=ints(start[at // 100] + at % 100), q=normal(rows, H * d), k=normal(rows, Hkv * d))
        s.update(q_out=torch.empty_like(s["q"]), k_out=torch.empty_like(s["k"]))
        return s
    B, page = case["B"], case["page"]
    n_rows = _lengths(case)
    used = [-(-n // page) for n in n_rows]
    if kind == "fork":
        # The sequences, then each one's beams; every fourth sequence has none and is given room instead.
        beams, room, n_pages = case["beams"], case["room"], _fork_pages(case)
        slots = B * (1 + beams)
        src = np.array([b for b in range(B) for _ in range(1 if b % 4 == 3 else beams)], np.int32)
        dst = np.array([b if b % 4 == 3 else B + b * beams + c for b in range(B) for c in range(1 if b % 4 == 3 else beams)], np.int32)
        rows = np.array(n_rows, np.int32)[src]
        keep = np.zeros(slots, np.int32)
        keep[:B] = n_rows
        order = rng.permutation(n_pages)
        stride = max(-(-(n + room) // page) for n in n_rows)
        table = np.full((slots, stride), -1, np.int32)
        refs = np.zeros(n_pages, np.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        refs[order[:at]] = 1
        refs[order[at:at + case["taken"]]] = rng.integers(1, 4, size=case["taken"])  # others'
        s.update(src=src, dst=dst, rows=rows, room=(rows + room).astype(np.int32), keep=keep, pairs=ints(np.full((len(src), 2), -1)),
                 missing=ints([-1]))
    elif kind == "compact":
        live, moves = sum(used), case["moves"]
        n_pages, stride = live + case["spare"], max(used)
        there = np.ones(live, bool)
        there[rng.permutation(live)[:moves]] = False
        behind = live + rng.permutation(case["spare"])[:moves]
        order = rng.permutation(np.concatenate((np.nonzero(there)[0], behind)))
        table = np.full((B, stride), -1, np.int32)
        refs = np.zeros(n_pages, np.int32)
        refs[order] = 1
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        if B > 1:  # the last sequence goes on from the first one's beginning as well
            both = min(used[0], used[-1]) // 2
            refs[table[-1, :both]], refs[table[0, :both]] = 1, 2
            table[-1, :both] = table[0, :both]
        s.update(table_out=ints(np.full_like(table, -7)), refs_out=ints(np.full_like(refs, -7)), moved=ints([-1, -1]),
                 pairs=ints(np.full((max(1, min(live, case["spare"])), 2), -1)))
    else:
        n_pages, stride = sum(used) + 2, max(used)
        order = rng.permutation(n_pages)
        table = np.full((B, stride), -1, np.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        refs = np.zeros(n_pages, np.int32)
        count = _nodes(case)
        q_start = np.cumsum([0] + count, dtype=np.int32)
        N, words = int(q_start[-1]), (max(count) + 63) // 64
        # Trees that are wide near their first token; a few tokens follow the cache's last row like it.
        parent, mask, path, kept = np.empty(N, np.int32), np.zeros((N, words), np.uint64), np.full(N, -1, np.int32), np.ones(B, np.int32)
        for b, n in enumerate(count):
            t0 = q_start[b]
            up = np.floor(rng.random(n) ** 1.5 * np.arange(n)).astype(np.int32)
            up[rng.random(n) < 0.03] = -1
            up[0] = -1
            parent[t0:t0 + n] = up
            depth = np.zeros(n, np.int32)
            for i in range(n):
                if up[i] >= 0:
                    mask[t0 + i] = mask[t0 + up[i]]
                    depth[i] = depth[up[i]] + 1
                mask[t0 + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
            # What was accepted: the way to a deep token, as far as a second pass over the same rows finds them unmoved.
            way, i = [], int(rng.choice(np.nonzero(depth >= min(depth.max(), 5))[0]))
            while i >= 0:
                way.insert(0, i)
                i = int(up[i])
            while any(p != j and p < len(way) for j, p in enumerate(way)):
                way.pop()
            path[t0:t0 + len(way)] = way
            kept[b] = len(way)
        s.update(q_start=q_start, N=N, words=words, parent=ints(parent), path=ints(path), kept=ints(kept))
        s["mask"] = torch.from_numpy(mask.view(np.int64)).cuda()
    s.update(n_rows=np.array(n_rows, dtype=np.int32), n_pages=n_pages, table=ints(table), refs=ints(refs))
    s.update(k=normal(n_pages, page, Hkv * d), v=normal(n_pages, page, Hkv * d))
    if kind in ("tree", "append"):
        s["q"] = normal(s["N"], case["H"] * d)
    if kind == "tree":
        s.update(out=torch.empty_like(s["q"]), lse=torch.empty(s["N"], case["H"], device="cuda"))
    if kind == "append":
        s.update(k_new=normal(s["N"], Hkv * d), v_new=normal(s["N"], Hkv * d), q_out=torch.empty_like(s["q"]),
                 mask=torch.zeros_like(s["mask"]), pos=torch.zeros(s["N"], device="cuda", dtype=torch.int32))
        # Positions run on after an eviction: they are past the rows.
        s["first"] = np.array([n - q + 1000 * (i % 3) for i, (n, q) in enumerate(zip(n_rows, count))], dtype=np.int32)
    return s


def _padded(s):
    """(token of each sequence's padded slot, whether the slot is one, rows of each sequence, row of each slot)."""
    q_start = torch.from_numpy(s["q_start"]).cuda().long()
    n_rows = torch.from_numpy(s["n_rows"]).cuda().long()
    q_len = q_start[1:] - q_start[:-1]
    i = torch.arange(int((s["q_start"][1:] - s["q_start"][:-1]).max()), device="cuda")
    is_token = i[None, :] < q_len[:, None]
    token = torch.where(is_token, q_start[:-1, None] + i[None, :], 0)
    return token, is_token, n_rows, (n_rows - q_len)[:, None] + i[None, :]


def _frequencies(case):
    """Angle per position of each pair, in 64 bits."""
    rot, scale = case["rot"], case["scale"]
    theta = THETA * FACTOR ** (rot / (rot - 2)) if scale == "base" else THETA
    f = theta ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / -rot)
    if scale == "linear":
        return f / FACTOR
    if scale == "turns":
        part = ((CONTEXT * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        return f * (part + (1 - part) / FACTOR)
    return f


def _amplitude(case):
    return AMPLITUDE if case["scale"] == "turns" else 1.0


def _turned(x, heads, case, pos, back=False):
    """x [N, heads * d] turned to its rows' positions; angles, and the turn itself, in 64 bits."""
    d, rot = case["d"], case["rot"]
    angle = pos.double()[:, None] * _frequencies(case)[None, :]
    c, sn = torch.cos(angle)[:, None, :] * _amplitude(case), torch.sin(angle)[:, None, :] * _amplitude(case)
    sn = -sn if back else sn
    y = x.view(-1, heads, d)
    z = y[..., :rot].double()
    lo, hi = (z[..., 0::2], z[..., 1::2]) if case["inter"] else (z[..., :rot // 2], z[..., rot // 2:])
    z = torch.stack((lo * c - hi * sn, hi * c + lo * sn), -1 if case["inter"] else -2).reshape(-1, heads, rot)
    return torch.cat((z.float(), y[..., rot:]), -1).view(-1, heads * d)


def _plain_turn(s):
    case = s["case"]
    return dict(q=_turned(s["q"], case["H"], case, s["pos"], case["back"]), k=_turned(s["k"], case["Hkv"], case, s["pos"], case["back"]))


def _plain_append(s):
    case = s["case"]
    H, Hkv, d, page = case["H"], case["Hkv"], case["d"], case["page"]
    token, is_token, _, row = _padded(s)
    B, T = token.shape
    # Who is above whom: steps up are doubled until they reach past the deepest.
    up = torch.where(is_token, s["parent"].long()[token], -1)
    me = torch.arange(T, device="cuda")
    step = torch.cat((torch.where(up < 0, T, up), torch.full((B, 1), T, device="cuda")), 1)
    sees = torch.zeros(B, T + 1, T + 1, device="cuda")
    sees[:, me, me] = 1
    for _ in range(T.bit_length()):
        # (ancestors within 2^k steps, then those of the one 2^k steps up)
        sees = ((sees + sees.gather(1, step[:, :, None].expand(-1, -1, T + 1))) > 0).float()
        step = step.gather(1, step)
    sees = sees[:, :T, :T]
    pos = (torch.from_numpy(s["first"]).cuda().long()[:, None] + sees.sum(-1).long() - 1)[is_token]
    bits = torch.nn.functional.pad(sees, (0, 64 * s["words"] - T)).long().view(B, T, s["words"], 64)
    mask = (bits << torch.arange(64, device="cuda")).sum(-1)[is_token]
    b = torch.arange(B, device="cuda")[:, None].expand_as(row)[is_token]
    row = row[is_token]
    at = s["table"][b, row // page].long() * page + row % page
    s["k"].view(-1, Hkv * d)[at] = _turned(s["k_new"], Hkv, case, pos)
    s["v"].view(-1, Hkv * d)[at] = s["v_new"]
    return dict(q=_turned(s["q"], H, case, pos), k=s["k"], v=s["v"], mask=mask, pos=pos.int())


def _plain_tree(s):
    case = s["case"]
    B, H, Hkv, d, page = case["B"], case["H"], case["Hkv"], case["d"], case["page"]
    g = H // Hkv
    token, is_token, n_rows, row = _padded(s)
    T, S = token.shape[1], int(s["n_rows"].max())
    at = torch.arange(S, device="cuda")
    rows = (s["table"][:, at // page].long() * page + at % page).clamp_(min=0)
    k = s["k"].view(-1, Hkv, d)[rows].permute(0, 2, 3, 1).contiguous().view(B * Hkv, d, S)
    v = s["v"].view(-1, Hkv, d)[rows].permute(0, 2, 1, 3).contiguous().view(B * Hkv, S, d)
    q = s["q"].view(-1, Hkv, g, d)[token].permute(0, 2, 3, 1, 4).contiguous().view(B * Hkv, g * T, d)
    score = torch.matmul(q, k).view(B, Hkv, g, T, S).mul_(1.0 / math.sqrt(d))
    new = at[None, :] - row[:, :1]  # a row's number among the new tokens
    of = new.clamp(0, 64 * s["words"] - 1)
    bit = (s["mask"][token].gather(2, (of // 64)[:, None, :].expand(B, T, S)) >> (of % 64)[:, None, :]) & 1
    sees = (new < 0)[:, None, :] | ((bit == 1) & (at[None, None, :] < n_rows[:, None, None]))
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total)
    o = torch.matmul(p.view(B * Hkv, g * T, S), v).view(B, Hkv, g, T, d)
    out = o.permute(0, 3, 1, 2, 4)[is_token].reshape(-1, H * d)
    return dict(out=out, lse=(top + total.log()).view(B, H, T).permute(0, 2, 1)[is_token])


def _plain_keep(s):
    case = s["case"]
    Hkv, d, page = case["Hkv"], case["d"], case["page"]
    token, is_token, _, row = _padded(s)
    number = torch.arange(token.shape[1], device="cuda")[None, :]
    moves = is_token & (number < s["kept"][:, None])
    b = torch.arange(case["B"], device="cuda")[:, None].expand_as(row)[moves]
    to, of = row[moves], (row[:, :1] + s["path"].long()[token])[moves]
    to = s["table"][b, to // page].long() * page + to % page
    of = s["table"][b, of // page].long() * page + of % page
    k, v = s["k"].view(-1, Hkv * d), s["v"].view(-1, Hkv * d)
    k[to] = k[of]
    v[to] = v[of]
    return dict(k=s["k"], v=s["v"])


def _plain_fork(s):
    table, refs, page = s["table"], s["refs"], s["case"]["page"]
    src, dst, rows, room, keep = (torch.from_numpy(s[x]).cuda().long() for x in ("src", "dst", "rows", "room", "keep"))
    at = torch.arange(table.shape[1], device="cuda")[None, :]
    gone = (at >= (keep[:, None] + page - 1) // page) & (table >= 0)
    refs.index_add_(0, table[gone].long(), torch.full((int(gone.sum()),), -1, device="cuda", dtype=torch.int32))
    table[gone] = -1
    # A page that is shared, one that is there already, and those that are wanted.
    of, self = table[src].long(), (src == dst)[:, None]
    whole, want = rows[:, None] // page, (room[:, None] + page - 1) // page
    shared = (at < whole) & ~self
    there = self & (of >= 0) & (refs[of.clamp(min=0)] == 1)
    fresh = (at >= whole) & (at < want) & ~there
    free = torch.nonzero(refs == 0)[:, 0]
    short = int(fresh.sum()) - free.numel()
    s["pairs"].fill_(-1)
    s["missing"].fill_(max(0, short))
    if short <= 0:
        page_of = torch.where(fresh, free[(fresh.flatten().cumsum(0) - 1).clamp(min=0)].view_as(of) if free.numel() else -1, of)
        refs.index_add_(0, of[shared], torch.ones(int(shared.sum()), device="cuda", dtype=torch.int32))
        left = fresh & self & (of >= 0)
        refs.index_add_(0, of[left], torch.full((int(left.sum()),), -1, device="cuda", dtype=torch.int32))
        refs[page_of[fresh]] = 1
        copied = fresh & (at == whole) & (rows[:, None] % page > 0)
        s["pairs"][copied.any(1)] = torch.stack((of[copied], page_of[copied]), 1).int()
        table[dst] = torch.where(at < want, page_of, torch.where(self, of, -1)).int()
        s["k"][page_of[copied]] = s["k"][of[copied]]
        s["v"][page_of[copied]] = s["v"][of[copied]]
    return dict(table=table, refs=refs, pairs=s["pairs"], missing=s["missing"], k=s["k"], v=s["v"])


def _plain_compact(s):
    refs, n = s["refs"], s["n_pages"]
    at = torch.arange(n, device="cuda")
    live = int((refs > 0).sum())
    to = torch.nonzero((refs == 0) & (at < live))[:, 0]
    of = torch.nonzero((refs > 0) & (at >= live))[:, 0].flip(0)
    m = min(len(to), s["pairs"].shape[0])
    goes = at.clone()
    goes[of[:m]] = to[:m]
    s["moved"][0], s["moved"][1] = m, len(to) - m
    s["pairs"].fill_(-1)
    s["pairs"][:m, 0], s["pairs"][:m, 1] = of[:m].int(), to[:m].int()
    s["table_out"].copy_(torch.where(s["table"] >= 0, goes[s["table"].long().clamp(min=0)], s["table"]))
    s["refs_out"].copy_(refs)
    s["refs_out"][to[:m]] = refs[of[:m]]
    s["refs_out"][of[:m]] = 0
    s["k"][to[:m]] = s["k"][of[:m]]
    s["v"][to[:m]] = s["v"][of[:m]]
    return dict(table=s["table_out"], refs=s["refs_out"], pairs=s["pairs"], moved=s["moved"], k=s["k"], v=s["v"])


_PLAIN = dict(turn=_plain_turn, append=_plain_append, tree=_plain_tree, keep=_plain_keep, fork=_plain_fork, compact=_plain_compact)
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


def _own_turns(s, L):
    """The host's frequencies, which a program keeps, and how they are used."""
    case = s["case"]
    if s["freq"] is None:
        s["freq"] = np.empty(case["rot"] // 2, np.float64)
        _done(L.zt_rope_frequencies(s["freq"].ctypes.data, case["rot"], THETA, SCALES.index(case["scale"]), FACTOR, LOW, HIGH, CONTEXT))
    return s["freq"].ctypes.data, case["rot"], int(case["inter"]), _amplitude(case)


def _own_workspace(s, nbytes):
    if s["ws"] is None:  # a serving program keeps one
        s["ws"] = torch.empty(max(nbytes, 16), device="cuda", dtype=torch.uint8)
    return s["ws"].data_ptr(), s["ws"].numel()


def _own_run(s):
    L, case = _lib(), s["case"]
    kind, Hkv, d = case["kind"], case["Hkv"], case["d"]
    stream = torch.cuda.current_stream().cuda_stream
    if kind == "turn":
        freq, rot, inter, amplitude = _own_turns(s, L)
        fn = L.zt_rope_at_backward if case["back"] else L.zt_rope_at_forward
        _done(fn(s["q"].data_ptr(), s["k"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(), s["pos"].data_ptr(),
                 freq, case["rows"], case["H"], Hkv, d, rot, inter, amplitude, stream))
        return dict(q=s["q_out"], k=s["k_out"])
    page, table, stride, n_pages = case["page"], s["table"].data_ptr(), s["table"].shape[1], s["n_pages"]
    k, v = s["k"].data_ptr(), s["v"].data_ptr()
    if kind == "fork":
        slots, n, rows, room = s["table"].shape[0], len(s["src"]), s["rows"].ctypes.data, s["room"].ctypes.data
        refs, pairs = s["refs"].data_ptr(), s["pairs"].data_ptr()
        ws, nbytes = _own_workspace(s, L.zt_paged_fork_workspace(rows, room, n, n_pages, page) if s["ws"] is None else 0)
        _done(L.zt_paged_free(table, refs, s["keep"].ctypes.data, slots, n_pages, page, stride, stream))
        _done(L.zt_paged_fork(table, refs, pairs, s["missing"].data_ptr(), s["src"].ctypes.data, s["dst"].ctypes.data, rows,
                              room, n, slots, n_pages, page, stride, ws, nbytes, stream))
        _done(L.zt_paged_copy(k, v, pairs, n, n_pages, page, Hkv, d, stream))
        return dict(table=s["table"], refs=s["refs"], pairs=s["pairs"], missing=s["missing"], k=s["k"], v=s["v"])
    if kind == "compact":
        pairs, most = s["pairs"].data_ptr(), s["pairs"].shape[0]
        ws, nbytes = _own_workspace(s, L.zt_paged_compact_workspace(n_pages) if s["ws"] is None else 0)
        _done(L.zt_paged_compact(table, s["refs"].data_ptr(), s["table_out"].data_ptr(), s["refs_out"].data_ptr(), pairs,
                                 s["moved"].data_ptr(), most, case["B"], n_pages, stride, ws, nbytes, stream))
        _done(L.zt_paged_copy(k, v, pairs, most, n_pages, page, Hkv, d, stream))
        return dict(table=s["table_out"], refs=s["refs_out"], pairs=s["pairs"], moved=s["moved"], k=s["k"], v=s["v"])
    B, q_start, n_rows = case["B"], s["q_start"].ctypes.data, s["n_rows"].ctypes.data
    if kind == "keep":
        _done(L.zt_paged_keep(k, v, table, s["path"].data_ptr(), s["kept"].data_ptr(), q_start, n_rows, B, n_pages, page,
                              stride, Hkv, d, stream))
        return dict(k=s["k"], v=s["v"])
    H = case["H"]
    if kind == "append":
        freq, rot, inter, amplitude = _own_turns(s, L)
        _done(L.zt_tree_mask(s["parent"].data_ptr(), s["mask"].data_ptr(), s["pos"].data_ptr(), q_start,
                             s["first"].ctypes.data, B, s["words"], stream))
        _done(L.zt_paged_append_at(s["q"].data_ptr(), s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["q_out"].data_ptr(), k,
                                   v, table, None, s["pos"].data_ptr(), freq, q_start, n_rows, B, n_pages, page, stride, 0,
                                   H, Hkv, d, rot, inter, amplitude, stream))
        return dict(q=s["q_out"], k=s["k"], v=s["v"], mask=s["mask"], pos=s["pos"])
    ws, nbytes = _own_workspace(s, L.zt_attn_paged_workspace(q_start, n_rows, B, H, Hkv, d, 0) if s["ws"] is None else 0)
    _done(L.zt_attn_paged_tree(s["q"].data_ptr(), k, v, table, s["mask"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(),
                               q_start, n_rows, B, n_pages, page, stride, s["words"], H, Hkv, d, ws, nbytes, stream))
    return dict(out=s["out"], lse=s["lse"])


def run(state):
    return _own_run(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    kind, Hkv, d = case["kind"], case["Hkv"], case["d"]
    if kind == "turn":
        n = case["rows"] * (case["H"] + Hkv)
        return dict(bytes=8 * n * d + 4 * case["rows"], flops=3 * n * case["rot"])
    n_rows, page = _lengths(case), case["page"]
    of_page = 4 * page * Hkv * d
    if kind == "fork":
        n, room, beams = n_rows, case["room"], case["beams"]
        tables = sum(-(-(x + room) // page) * (1 if b % 4 == 3 else beams) for b, x in enumerate(n))
        tails = sum(beams for b, x in enumerate(n) if b % 4 != 3 and x % page)
        # The counts read; the tables' entries read, written and dropped, with a count each; a page of K and V for each beam.
        return dict(bytes=4 * _fork_pages(case) + 20 * tables + 4 * of_page * tails, flops=0)
    if kind == "compact":
        pages = sum(-(-x // page) for x in n_rows)
        # Tables and counts read and written; the moved pages of K and V.
        return dict(bytes=8 * (2 * pages + case["spare"]) + 4 * of_page * case["moves"], flops=0)
    q_len = _nodes(case)
    N, words = sum(q_len), (max(q_len) + 63) // 64
    if kind == "keep":
        # About five rows of each tree are kept; the first stays where it is.
        kept = sum(min(4, n - 1) for n in q_len)
        return dict(bytes=16 * kept * Hkv * d, flops=0)
    H = case["H"]
    if kind == "append":
        # q, k, v in; q out, k, v into the cache; parents in, masks and positions out.
        return dict(bytes=4 * N * (2 * H + 4 * Hkv) * d + N * (8 + 8 * words), flops=3 * N * (H + Hkv) * case["rot"])
    # q in, out and the log-sum-exp out, the K and V rows, the masks; a token sees about a tenth of its tree.
    seen = sum(n_rows)
    pairs = sum(q * (n - q) + q * (1 + q // 10) for n, q in zip(n_rows, q_len))
    return dict(bytes=4 * (2 * N * H * d + N * H + 2 * seen * Hkv * d) + 8 * N * words, flops=4 * H * d * pairs)


def exact(case, seed):
    x = prepare(case, seed)
    kind, Hkv, d = case["kind"], case["Hkv"], case["d"]

    def turned(rows, heads, pos, back=False):
        """Pairs as complex numbers times e^(i angle)."""
        rot = case["rot"]
        base = THETA * FACTOR ** (rot / (rot - 2)) if case["scale"] == "base" else THETA
        f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
        if case["scale"] == "linear":
            f = f / FACTOR
        if case["scale"] == "turns":
            for i, r in enumerate(CONTEXT * f / (2 * np.pi)):
                s = min(1.0, max(0.0, (r - LOW) / (HIGH - LOW)))
                f[i] = s * f[i] + (1 - s) * f[i] / FACTOR
        y = rows.double().view(-1, heads, d).clone()
        z = y[..., :rot]
        z = z.reshape(-1, heads, rot // 2, 2) if case["inter"] else z.reshape(-1, heads, 2, rot // 2).transpose(2, 3)
        angle = pos.double()[:, None, None] * torch.from_numpy(-f if back else f).cuda()
        z = torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(angle, _amplitude(case)), angle)
        z = torch.view_as_real(z)
        y[..., :rot] = z.reshape(-1, heads, rot) if case["inter"] else z.transpose(2, 3).reshape(-1, heads, rot)
        return y.view(-1, heads * d)

    if kind == "turn":
        return dict(q=turned(x["q"], case["H"], x["pos"], case["back"]), k=turned(x["k"], Hkv, x["pos"], case["back"]))
    page, n_rows = case["page"], x["n_rows"].tolist()
    table, refs = x["table"].cpu().numpy(), x["refs"].cpu().numpy()
    k, v = x["k"].double(), x["v"].double()

    def places(b, n):
        r = np.arange(n)
        return torch.from_numpy(table[b][r // page].astype(np.int64) * page + r % page).cuda()

    if kind == "fork":
        for b, n in enumerate(x["keep"].tolist()):
            for j in range(-(-n // page), table.shape[1]):
                if table[b, j] >= 0:
                    refs[table[b, j]] -= 1
                table[b, j] = -1
        before, free = refs.copy(), iter(np.nonzero(refs == 0)[0].tolist())
        pairs = np.full((len(x["src"]), 2), -1, np.int32)
        for i, (a, b, n, room) in enumerate(zip(*(x[y].tolist() for y in ("src", "dst", "rows", "room")))):
            for j in range(-(-room // page)):
                p = int(table[a, j])
                if j < n // page:
                    if a != b:
                        table[b, j] = p
                        refs[p] += 1
                    continue
                if a == b and p >= 0 and before[p] == 1:
                    continue
                table[b, j] = next(free)
                refs[table[b, j]] = 1
                if a == b and p >= 0:
                    refs[p] -= 1
                if j == n // page and n % page:
                    pairs[i] = p, table[b, j]
                    k[table[b, j]], v[table[b, j]] = k[p], v[p]
        return dict(table=torch.from_numpy(table).cuda(), refs=torch.from_numpy(refs).cuda(), pairs=torch.from_numpy(pairs).cuda(),
                    missing=torch.zeros(1, device="cuda", dtype=torch.int32), k=k, v=v)
    if kind == "compact":
        pairs = np.full(tuple(x["pairs"].shape), -1, np.int32)
        lo, hi, m = 0, len(refs) - 1, 0
        while True:
            while lo < len(refs) and refs[lo]:
                lo += 1
            while hi >= 0 and not refs[hi]:
                hi -= 1
            if lo >= hi:
                break
            pairs[m] = hi, lo
            refs[lo], refs[hi] = refs[hi], 0
            m += 1
        now = np.arange(len(refs), dtype=np.int32)
        now[pairs[:m, 0]] = pairs[:m, 1]
        table = np.where(table < 0, table, now[table])
        of, to = (torch.from_numpy(pairs[:m, i].astype(np.int64)).cuda() for i in range(2))
        k[to], v[to] = k[of], v[of]
        return dict(table=torch.from_numpy(table).cuda(), refs=torch.from_numpy(refs).cuda(), pairs=torch.from_numpy(pairs).cuda(),
                    moved=torch.tensor([m, 0], device="cuda", dtype=torch.int32), k=k, v=v)
    q_start, parent = x["q_start"].tolist(), x["parent"].cpu().numpy()
    kf, vf = k.view(-1, Hkv * d), v.view(-1, Hkv * d)
    if kind == "keep":
        path, kept = x["path"].cpu().numpy(), x["kept"].tolist()
        for b, n in enumerate(n_rows):
            at = places(b, n)[n - (q_start[b + 1] - q_start[b]):]
            way = torch.from_numpy(path[q_start[b]:q_start[b] + kept[b]].astype(np.int64)).cuda()
            kf[at[:kept[b]]], vf[at[:kept[b]]] = kf[at[way]], vf[at[way]]
        return dict(k=k, v=v)
    H = case["H"]
    # A token's line: itself and its ancestors.
    line = []
    for b in range(len(n_rows)):
        for i in range(q_start[b + 1] - q_start[b]):
            line.append(([] if parent[q_start[b] + i] < 0 else line[q_start[b] + parent[q_start[b] + i]]) + [i])
    if kind == "append":
        mask = np.zeros((x["N"], x["words"]), np.uint64)
        pos = np.empty(x["N"], np.int32)
        for b, n in enumerate(n_rows):
            for t in range(q_start[b], q_start[b + 1]):
                pos[t] = x["first"][b] + len(line[t]) - 1
                for j in line[t]:
                    mask[t, j // 64] |= np.uint64(1 << (j % 64))
        pos_d = torch.from_numpy(pos).cuda()
        k_new, q = turned(x["k_new"], Hkv, pos_d), turned(x["q"], H, pos_d)
        for b, n in enumerate(n_rows):
            at = places(b, n)[n - (q_start[b + 1] - q_start[b]):]
            kf[at], vf[at] = k_new[q_start[b]:q_start[b + 1]], x["v_new"][q_start[b]:q_start[b + 1]].double()
        return dict(q=q, k=k, v=v, mask=torch.from_numpy(mask.view(np.int64)).cuda(), pos=pos_d)
    g = H // Hkv
    out = torch.empty(x["N"], H, d, device="cuda", dtype=torch.float64)
    lse = torch.empty(x["N"], H, device="cuda", dtype=torch.float64)
    q = x["q"].view(-1, H, d)
    for b, n in enumerate(n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        sees = np.zeros((t1 - t0, n), bool)
        sees[:, :n - (t1 - t0)] = True
        for t in range(t0, t1):
            sees[t - t0, [n - (t1 - t0) + j for j in line[t]]] = True
        hidden, at = ~torch.from_numpy(sees).cuda(), places(b, n)
        for j in range(Hkv):
            kk, vv = (y.view(-1, Hkv, d)[at, j].contiguous() for y in (kf, vf))
            for h in range(j * g, (j + 1) * g):
                score = (q[t0:t1, h].double() @ kk.t().contiguous()) / math.sqrt(d)
                score = score.masked_fill(hidden, -math.inf)
                lse[t0:t1, h] = torch.logsumexp(score, 1)
                out[t0:t1, h] = torch.softmax(score, 1) @ vv
    return dict(out=out.view(-1, H * d), lse=lse)
