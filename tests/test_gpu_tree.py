"""Trees of drafted tokens, rotary positions and shared pages on the GPU against treeref (64 bits), and a serving run of all
of them."""
import numpy as np
import pytest

import pagedref
import treeref
from test_gpu_paged import Cache, grade

pytestmark = pytest.mark.gpu
EPS = pagedref.EPS


def dev(gpu, x):
    x = np.ascontiguousarray(x)
    return gpu.from_numpy(x.view(np.int64) if x.dtype == np.uint64 else x).cuda()


def run_tree(gpu, zt, c, q_h, mask_h, q_start, H, lse=True, stream=None):
    """out and lse; rows that no token has, and the workspace, begin as NaN."""
    q, mask = dev(gpu, np.asarray(q_h, np.float32)), dev(gpu, mask_h)
    out = gpu.full_like(q, float("nan"))
    l = gpu.full(q.shape[:2], float("nan"), device="cuda") if lse else None
    need = zt.attn_paged_workspace_bytes(q_start, c.n_rows, H, c.Hkv, c.d)
    ws = gpu.full((need // 4,), float("nan"), device="cuda") if need else None
    if stream is not None:
        stream.wait_stream(gpu.cuda.current_stream())
    zt.attn_paged_tree(q, c.k, c.v, c.table, mask, out, q_start, c.n_rows, c.page, H, c.Hkv, c.d, ws, l, stream)
    gpu.cuda.synchronize()
    return out.cpu().numpy(), None if l is None else l.cpu().numpy(), None


def reference(c, q, mask, q_start, H):
    sees = [treeref.seen(mask[q_start[b]:q_start[b + 1]], n, q_start[b + 1] - q_start[b]) for b, n in enumerate(c.n_rows)]
    out, lse, bound = treeref.attend(q, c.k_h, c.v_h, c.table_h, q_start, c.n_rows, c.page, H, c.Hkv, c.d, sees)
    return out, lse, None, bound, None


def check(got, ref, q_start):
    """grade(), and exactly 0 and -inf where a token sees nothing."""
    none = np.isneginf(ref[1])
    rows = slice(q_start[0], q_start[-1])
    assert np.all(got[0][rows][none[rows]] == 0)
    if got[1] is not None:
        assert np.all(np.isneginf(got[1][rows]) == none[rows])
        ref[1][none] = 0  # (graded above)
        got[1][none & (np.arange(len(none)) >= q_start[0])[:, None] & (np.arange(len(none)) < q_start[-1])[:, None]] = 0
    grade(got, ref, q_start, None, None)


SHAPES = [(4, 2, 32), (8, 8, 64), (6, 2, 64), (32, 8, 128), (8, 2, 96), (16, 4, 256), (5, 1, 128), (2, 1, 160), (4, 4, 34),
          (6, 3, 50), (9, 3, 250), (4, 1, 192), (64, 1, 64), (33, 1, 32)]
# (rows with the new tokens, new tokens): trees of one token and none, no rows before them, ends inside a tile and at it.
BATCHES = {
    "single_tokens": ([1, 2, 16, 17, 33, 200], [1] * 6),
    "drafts": ([40, 0, 7, 64, 129, 31, 500], [3, 0, 7, 0, 17, 31, 5]),
    "wide": ([333, 64, 700], [90, 64, 26]),
    "words": ([150, 260], [150, 129]),
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("H,Hkv,d", SHAPES)
@pytest.mark.parametrize("any_mask", [False, True])
def test_attention(gpu, zt, H, Hkv, d, page, batch, any_mask):
    """Trees, and masks of any bits (later tokens', past the last, empty ones) in words more than needed."""
    n_rows, q_len = BATCHES[batch]
    rng = np.random.default_rng([H, Hkv, d, page, len(n_rows), any_mask])
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([2] + q_len).tolist()  # the packed tokens begin behind two that are not this call's
    words = (max(q_len) + 63) // 64 + any_mask
    mask = np.full((q_start[-1] + 3, words), 2 ** 64 - 1, np.uint64)
    if any_mask:
        mask[:] = rng.integers(0, 2 ** 64, mask.shape, dtype=np.uint64)
        mask[rng.random(len(mask)) < 0.2] = 0
    else:
        mask[q_start[0]:q_start[-1]] = treeref.masks([treeref.random_tree(rng, n) for n in q_len], words)[0]
    q = rng.standard_normal((q_start[-1] + 3, H, d)).astype(np.float32)
    check(run_tree(gpu, zt, c, q, mask, q_start, H, lse=page != 16), reference(c, q, mask, q_start, H), q_start)


@pytest.mark.parametrize("H,Hkv,d", SHAPES)
def test_a_line_is_a_chunk(gpu, zt, H, Hkv, d):
    """Every token its successor's parent: zt_attn_paged's outputs, bit for bit."""
    n_rows, q_len, page = [300, 77, 9, 140, 33, 1, 2600, 4000], [1, 4, 8, 90, 33, 1, 130, 16], 16
    rng = np.random.default_rng([H, d])
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([0] + list(q_len)).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    mask = treeref.masks([np.arange(-1, n - 1) for n in q_len], 3)[0]
    out, lse, _ = run_tree(gpu, zt, c, q, mask, q_start, H)
    qd, o, l = dev(gpu, q), gpu.empty(q.shape, device="cuda"), gpu.empty(q.shape[:2], device="cuda")
    ws = gpu.empty(zt.attn_paged_workspace_bytes(q_start, n_rows, H, Hkv, d), device="cuda", dtype=gpu.uint8)
    zt.attn_paged(qd, c.k, c.v, c.table, o, q_start, n_rows, page, H, Hkv, d, ws, l)
    assert np.array_equal(o.cpu().numpy(), out) and np.array_equal(l.cpu().numpy(), lse)


@pytest.mark.parametrize("n,L", [(16, 16), (29, 29), (300, 17), (700, 26), (1021, 31)])
@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 64), (4, 1, 50), (8, 2, 96), (12, 3, 82), (32, 8, 128), (4, 1, 98)])
def test_a_small_grid_of_65_to_128_rows(gpu, zt, H, Hkv, d, n, L):
    """The shape that only trees have (five to eight blocks of 16 rows, one chunk or several), with a value past 2^40 and one
    that is not finite in rows of the tree that some tokens do not see."""
    rng = np.random.default_rng([H, d, n])
    c = Cache(gpu, rng, [n], 16, Hkv, d, garbage=np.nan)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    up = treeref.random_tree(rng, L)
    mask = treeref.masks([up], 1)[0]
    check(run_tree(gpu, zt, c, q, mask, [0, L], H), reference(c, q, mask, [0, L], H), [0, L])
    at = pagedref.places(c.table_h, 0, n, 16)[n - L + L // 2]
    c.v_h[at, :, 1] = np.float32(2.0 ** 50)
    c.k_h[at, :, 2] = np.float32(2.0 ** 41)
    q[:, :, 2] = np.float32(2.0 ** -40)
    c.k, c.v = dev(gpu, c.k_h), dev(gpu, c.v_h)
    got, ref = run_tree(gpu, zt, c, q, mask, [0, L], H), reference(c, q, mask, [0, L], H)
    check(got, ref, [0, L])
    hit = np.array([L // 2 in line for line in treeref.lines(up)])
    before = run_tree(gpu, zt, c, q, mask, [0, L], H)
    c.v[at, :, 5] = float("nan")
    c.k[at, :, 7] = float("inf")
    after = run_tree(gpu, zt, c, q, mask, [0, L], H)
    assert hit.any() and not hit.all()
    assert np.array_equal(before[0][~hit], after[0][~hit]) and np.array_equal(before[1][~hit], after[1][~hit])
    assert np.all(np.isnan(after[0][hit][..., 5]))


def test_a_long_line(gpu, zt):
    """A tree of 1500 tokens that is a line, as long as its cache and behind other rows: the chunk's outputs, bit for bit."""
    H, Hkv, d, page, n_rows, q_len = 8, 2, 128, 16, [1500, 1703], [1500, 1500]
    rng = np.random.default_rng(12)
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    q = gpu.randn(3000, H, d, device="cuda")
    mask, parent = gpu.empty(3000, 24, device="cuda", dtype=gpu.int64), np.tile(np.arange(-1, 1499, dtype=np.int32), 2)
    zt.tree_mask(dev(gpu, parent), mask, [0, 1500, 3000])
    got, want = gpu.empty_like(q), gpu.empty_like(q)
    ws = gpu.empty(zt.attn_paged_workspace_bytes([0, 1500, 3000], n_rows, H, Hkv, d) + 16, device="cuda", dtype=gpu.uint8)
    zt.attn_paged_tree(q, c.k, c.v, c.table, mask, got, [0, 1500, 3000], n_rows, page, H, Hkv, d, ws)
    zt.attn_paged(q, c.k, c.v, c.table, want, [0, 1500, 3000], n_rows, page, H, Hkv, d, ws)
    assert gpu.equal(got, want)


def test_no_tokens(gpu, zt):
    """Sequences without new tokens: nothing is written."""
    table, i32 = gpu.zeros(2, 4, device="cuda", dtype=gpu.int32), dict(device="cuda", dtype=gpu.int32)
    k, v, q = (gpu.full((4, 8, 32), 7.0, device="cuda") for _ in range(3))
    mask, pos = gpu.full((2, 1), 7, device="cuda", dtype=gpu.int64), gpu.full((2,), 7, **i32)
    zt.tree_mask(pos, mask, [0, 0, 0], pos, [1, 2])
    zt.attn_paged_tree(q, k, v, table, mask, q, [0, 0, 0], [5, 0], 8, 1, 1, 32, None)
    zt.paged_append_at(q, k, v, q, k, v, table, pos, zt.rope_frequencies(32), [0, 0, 0], [5, 0], 8, 1, 1, 32, 32)
    zt.paged_keep(k, v, table, pos, pos, [0, 0, 0], [5, 0], 8, 1, 32)
    zt.paged_copy(k, v, gpu.empty(0, 2, **i32), 8, 1, 32)
    assert all(bool((x == 7).all()) for x in (k, v, q, mask, pos))


@pytest.mark.parametrize("wgs", [256, 32768])
@pytest.mark.parametrize("H,Hkv,d,rows", pagedref.FEW_SHAPES)
def test_forced_chunk_counts(gpu, zt, tune, H, Hkv, d, rows, wgs):
    n_rows, q_len = pagedref.batch_of_few(H, Hkv, rows)
    rng = np.random.default_rng([H, d, rows])
    c = Cache(gpu, rng, n_rows, 16, Hkv, d)
    q_start = np.cumsum([0] + list(q_len)).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    mask = treeref.masks([treeref.random_tree(rng, n, 3.0) for n in q_len], 1)[0]
    tune({"ZT_PAGED_WGS": wgs})
    check(run_tree(gpu, zt, c, q, mask, q_start, H), reference(c, q, mask, q_start, H), q_start)


@pytest.mark.parametrize("H,Hkv,d", [(8, 8, 32), (16, 8, 64), (32, 8, 128), (16, 8, 256)])
def test_a_batch_of_every_kind(gpu, zt, H, Hkv, d):
    """More sequences than a launch takes, and launches of every kind beside one another."""
    n_rows, q_len = pagedref.batch_of_kinds(H, Hkv)
    rng = np.random.default_rng([H, d, 1])
    c = Cache(gpu, rng, n_rows, 16, Hkv, d)
    q_start = np.cumsum([0] + list(q_len)).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    mask = treeref.masks([treeref.random_tree(rng, n) for n in q_len], (max(q_len) + 63) // 64)[0]
    check(run_tree(gpu, zt, c, q, mask, q_start, H), reference(c, q, mask, q_start, H), q_start)


@pytest.mark.parametrize("L", [6, 30, 150])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 128), (6, 2, 50), (4, 1, 256), (4, 1, 192)])
def test_nothing_before_the_tree(gpu, zt, H, Hkv, d, L):
    """A cache of the new tokens alone: some see nothing, among them the first, and tokens that see only what is behind
    them; V's first row is not finite."""
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [L], 8, Hkv, d, garbage=np.nan)
    mask = treeref.masks([treeref.random_tree(rng, L)], (L + 63) // 64)[0]
    mask[::3] = 0
    mask[3::6, -1] = np.uint64(1) << np.uint64((L - 1) % 64)
    mask[1:, 0] &= ~np.uint64(1)
    c.v_h[pagedref.places(c.table_h, 0, 1, 8)] = np.inf
    c.v = dev(gpu, c.v_h)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    c.v_h[pagedref.places(c.table_h, 0, 1, 8)] = 0  # (which no token sees)
    check(run_tree(gpu, zt, c, q, mask, [0, L], H), reference(c, q, mask, [0, L], H), [0, L])


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("L,n", [(9, 40), (70, 130), (70, 70), (150, 1500)])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 128), (6, 2, 50), (4, 1, 256), (8, 2, 96)])
def test_what_a_token_does_not_see_changes_nothing(gpu, zt, H, Hkv, d, L, n, value):
    """K and V of one token in the tree's middle not finite: tokens of other lines as without, bit for bit."""
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [n], 16, Hkv, d)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    up = treeref.random_tree(rng, L)
    at = L // 3
    mask = treeref.masks([up], (L + 63) // 64)[0]
    hit = np.array([at in line for line in treeref.lines(up)])
    assert hit.any() and not hit.all()
    out0, lse0, _ = run_tree(gpu, zt, c, q, mask, [0, L], H)
    row = pagedref.places(c.table_h, 0, n, 16)[n - L + at]
    c.v[row, :, 3] = float(value)
    out1, lse1, _ = run_tree(gpu, zt, c, q, mask, [0, L], H)
    keep = np.arange(d) != 3
    assert np.array_equal(out0[~hit], out1[~hit]) and np.array_equal(lse0, lse1)
    assert np.array_equal(out0[hit][..., keep], out1[hit][..., keep])
    assert np.all(np.isnan(out1[hit][..., 3]) if np.isnan(value) else out1[hit][..., 3] == value)
    c.k[row] = float(value)
    out2, lse2, _ = run_tree(gpu, zt, c, q, mask, [0, L], H)
    assert np.array_equal(out0[~hit], out2[~hit]) and np.array_equal(lse0[~hit], lse2[~hit])
    # inf * q over columns of both signs: NaN scores, and with them the token's whole row.
    assert np.all(np.isnan(out2[hit])) and np.all(np.isnan(lse2[hit]))


@pytest.mark.parametrize("L", [5, 40, 150])
@pytest.mark.parametrize("where", ["k", "q", "both", "v"])
@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 64), (8, 2, 128), (4, 1, 256), (6, 2, 50)])
def test_large_values(gpu, zt, H, Hkv, d, where, L):
    """Values past 2^40, which leave the split products, in rows that some tokens see and others do not."""
    n, page = 220, 16
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [n], page, Hkv, d)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    big, some = np.float32(2.0 ** 45), rng.random(c.k_h.shape[0]) < 0.1
    if where in ("k", "both"):
        c.k_h[some, :, 5] *= big
        q[:, :, 5] /= big
    if where in ("q", "both"):
        q[::3, :, d - 2] *= big
        c.k_h[:, :, d - 2] /= big
    if where == "v":
        c.v_h[some, :, 7] *= big
    c.k, c.v = dev(gpu, c.k_h), dev(gpu, c.v_h)
    mask = treeref.masks([treeref.random_tree(rng, L)], 3)[0]
    check(run_tree(gpu, zt, c, q, mask, [0, L], H), reference(c, q, mask, [0, L], H), [0, L])


@pytest.mark.parametrize("bad", [-1, -(2 ** 31), 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("L", [9, 70])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 128), (4, 1, 256)])
def test_a_key_without_a_page(gpu, zt, H, Hkv, d, L, bad):
    """A page of new tokens that is none of the pool's: NaN for those that see one of its keys, the others as without."""
    n, page = 131, 4
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [n], page, Hkv, d)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    up = treeref.random_tree(rng, L)
    mask = treeref.masks([up], 2)[0]
    at = (n - L // 2) // page
    gone = set(range(at * page - (n - L), at * page + page - (n - L)))
    hit = np.array([bool(gone & set(line)) for line in treeref.lines(up)])
    assert hit.any() and not hit.all()
    out0, lse0, _ = run_tree(gpu, zt, c, q, mask, [0, L], H)
    c.table[0, at] = bad
    out1, lse1, _ = run_tree(gpu, zt, c, q, mask, [0, L], H)
    assert np.array_equal(out0[~hit], out1[~hit]) and np.array_equal(lse0[~hit], lse1[~hit])
    assert np.all(np.isnan(out1[hit])) and np.all(np.isnan(lse1[hit]))


@pytest.mark.parametrize("lengths", [[1], [0, 5, 64, 65, 0, 200, 256, 257], [4096, 300], [4500], [3] * 150])
def test_masks(gpu, zt, lengths):
    """Trees, and among their parents numbers that are no earlier token's; masks of more words than needed."""
    rng = np.random.default_rng(len(lengths))
    parents = []
    for n in lengths:
        up = treeref.random_tree(rng, n, 0.7)
        if n > 4:
            up[rng.integers(1, n, 3)] = [n, -5, 2 ** 31 - 1]
            i = int(rng.integers(1, n))
            up[i] = i  # itself
        parents.append(up)
    if lengths == [4500]:
        parents = [np.arange(-1, 4499, dtype=np.int32)]  # one line, past what LDS holds
    words = (max(lengths) + 63) // 64 + 1
    q_start = np.cumsum([3] + lengths)
    N = int(q_start[-1])
    parent, mask = np.full(N + 2, 77, np.int32), gpu.full((N + 2, words), -3, device="cuda", dtype=gpu.int64)
    pos_out = gpu.full((N + 2,), -3, device="cuda", dtype=gpu.int32)
    parent[3:N] = np.concatenate(parents)
    pos = rng.integers(0, 10 ** 6, len(lengths))
    zt.tree_mask(dev(gpu, parent), mask, q_start, pos_out, pos)
    want, depth = treeref.masks(parents, words)
    got, at = mask.cpu().numpy(), pos_out.cpu().numpy()
    assert np.array_equal(got[3:N].view(np.uint64), want)
    assert np.array_equal(at[3:N], np.repeat(pos, lengths) + depth)
    assert np.all(got[:3] == -3) and np.all(got[N:] == -3) and np.all(at[:3] == -3) and np.all(at[N:] == -3)
    mask2 = gpu.full_like(mask, -3)
    zt.tree_mask(dev(gpu, parent), mask2, q_start)
    assert gpu.equal(mask, mask2)


# ---- rotary positions ----------------------------------------------------------------------

TURNS = [(128, 128), (128, 64), (128, 96), (64, 36), (50, 26), (34, 34), (256, 256), (256, 128), (96, 72), (2, 2), (6, 4), (250, 126)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", TURNS)
@pytest.mark.parametrize("rows,H,Hkv", [(1, 4, 2), (37, 12, 4), (700, 3, 1), (5, 1, 0), (5, 0, 3)])
def test_turns(gpu, zt, rows, H, Hkv, d, rot, inter):
    rng = np.random.default_rng([rows, d, rot, inter])
    q, k = rng.standard_normal((rows, H, d)).astype(np.float32), rng.standard_normal((rows, Hkv, d)).astype(np.float32)
    pos = rng.integers(-(2 ** 31) if rows == 37 else 0, 2 ** 31 - 1 if rows == 37 else 10 ** 5, rows).astype(np.int32)
    freq = zt.rope_frequencies(rot, 500000.0, zt.ZT_ROPE_TURNS, 8.0, 1.0, 4.0, 8192.0)
    for back in (False, True):
        for place in ("out", "in"):
            qd, kd = dev(gpu, q) if H else None, dev(gpu, k) if Hkv else None
            qo, ko = (qd, kd) if place == "in" else [None if x is None else gpu.full_like(x, float("nan")) for x in (qd, kd)]
            zt.rope_at(qd, kd, qo, ko, dev(gpu, pos), freq, H, Hkv, d, rot, inter, 1.25, back)
            for x, y in ((q, qo), (k, ko)):
                if y is None:
                    continue
                want, bound = treeref.turn(x, pos, freq, rot, inter, 1.25, back)
                got = y.cpu().numpy()
                assert np.all(np.abs(got - want) <= bound)
                assert np.array_equal(got[..., rot:], x[..., rot:])


def test_many_rows_and_a_q_in_place_beside_a_k_that_is_not(gpu, zt):
    rows, H, Hkv, d, rot = 20011, 4, 2, 64, 32
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((rows, H, d)).astype(np.float32), rng.standard_normal((rows, Hkv, d)).astype(np.float32)
    pos, freq = rng.integers(0, 10 ** 5, rows).astype(np.int32), zt.rope_frequencies(rot)
    qd, ko = dev(gpu, q), gpu.full(k.shape, float("nan"), device="cuda")
    zt.rope_at(qd, dev(gpu, k), qd, ko, dev(gpu, pos), freq, H, Hkv, d, rot)
    for x, y in ((q, qd), (k, ko)):
        want, bound = treeref.turn(x, pos, freq, rot, False)
        assert np.all(np.abs(y.cpu().numpy() - want) <= bound)


def test_more_rows_than_a_launch_takes(gpu, zt):
    """2^24 + 5 rows, of which a launch takes 2^24 - 1."""
    rows = (1 << 24) + 5
    x = gpu.randn(rows, 2, device="cuda")
    pos = gpu.arange(rows, device="cuda", dtype=gpu.int32)
    y = gpu.full_like(x, float("nan"))
    zt.rope_at(x, None, y, None, pos, [0.37], 1, 0, 2, 2)
    at = np.r_[0:3, 12345, rows - 9:rows]
    want, bound = treeref.turn(x[at].cpu().numpy()[:, None], at, [0.37], 2, False)
    assert np.all(np.abs(y[at].cpu().numpy()[:, None] - want) <= bound) and not bool(y.isnan().any())


def test_whole_heads_are_the_plain_rope(gpu, zt):
    """Positions in order, whole heads, unscaled: zt_rope_qk_forward's rows, whose angles are t / theta^e where these are
    t theta^-e (a few steps of 64 bits apart)."""
    T, H, Hkv, d = 300, 4, 2, 64
    rng = np.random.default_rng(2)
    q, k = dev(gpu, rng.standard_normal((T, H * d)).astype(np.float32)), dev(gpu, rng.standard_normal((T, Hkv * d)).astype(np.float32))
    pos = gpu.arange(7, 7 + T, device="cuda", dtype=gpu.int32)
    for back in (False, True):
        a, b, c, e = (gpu.empty_like(x) for x in (q, k, q, k))
        zt.rope_qk(q, k, a, b, 1, T, H, Hkv, d, 7, 500000.0, back)
        zt.rope_at(q, k, c, e, pos, zt.rope_frequencies(d), H, Hkv, d, d, backward=back)
        for x, y in ((a, c), (b, e)):
            assert ((x - y).abs() <= 2 * 2 * EPS * x.abs() + 1e-12).all()


@pytest.mark.parametrize("inter", [False, True])
def test_the_way_back_is_the_gradient(gpu, zt, inter):
    """d/dx <g, turn(x)> = back(g), by the formula's transpose and by differences (the turn is linear: a whole step is exact
    up to the roundings, three of 2^-24 of the terms)."""
    rows, H, Hkv, d, rot, amp = 11, 3, 1, 34, 20, 1.5
    rng = np.random.default_rng(5)
    pos, freq = rng.integers(0, 1000, rows).astype(np.int32), zt.rope_frequencies(rot, 1e4, zt.ZT_ROPE_BASE, 4.0)
    x, g = (rng.standard_normal((rows, H, d)).astype(np.float32) for _ in range(2))
    k = dev(gpu, np.zeros((rows, Hkv, d), np.float32))

    def turn(y, back=False):
        out = gpu.empty(y.shape, device="cuda")
        zt.rope_at(dev(gpu, y), k, out, gpu.empty_like(k), dev(gpu, pos), freq, H, Hkv, d, rot, inter, amp, back)
        return out.cpu().numpy().astype(np.float64)

    back = turn(g, True)
    lhs, rhs = (turn(x) * g).sum(-1), (back * x).sum(-1)
    assert np.all(np.abs(lhs - rhs) <= 4 * amp * EPS * (np.abs(x) @ np.ones(d)) * np.abs(g).max(-1))
    for i in (0, 1, rot // 2, rot - 1, rot, d - 1):
        step = x.copy()
        step[..., i] += np.float32(1)
        h = (step.astype(np.float64) - x)[..., i]
        slope = ((turn(step) - turn(x)) * g).sum(-1) / h
        # Each of the two (or one) columns that change is rounded in both turns.
        off = 2 * 2 * EPS * 2 * amp * (np.abs(x).max(-1) + 2) * np.abs(g).max(-1) / np.abs(h) + 2 * EPS * np.abs(back[..., i])
        assert np.all(np.abs(slope - back[..., i]) <= off)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("H,Hkv,d,rot", [(4, 2, 32, 32), (32, 8, 128, 128), (16, 4, 256, 128), (6, 3, 50, 26), (4, 4, 34, 34), (8, 2, 96, 72),
                                         (12, 4, 64, 36)])
@pytest.mark.parametrize("batch", ["drafts", "many", "one"])
def test_append_at(gpu, zt, H, Hkv, d, rot, inter, batch):
    rng = np.random.default_rng([H, d, rot, inter])
    n_rows, q_len = {"drafts": BATCHES["drafts"], "one": ([300], [61]),
                     "many": ([20 + i % 30 for i in range(150)], [i % 5 for i in range(150)])}[batch]
    page, B = 8, len(n_rows)
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    q_start = np.cumsum([1] + q_len).tolist()
    N = q_start[-1]
    q, kn, vn = (rng.standard_normal((N + 2, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
    pos = rng.integers(0, 10 ** 5, N + 2).astype(np.int32)
    freq = zt.rope_frequencies(rot, 1e4, zt.ZT_ROPE_LINEAR, 2.0)
    w = rng.random((B, Hkv, max(n_rows) + 3), np.float32)
    lost = [b for b in range(B) if q_len[b] > 2][:1]  # the last page of one sequence is none of the pool's
    for b in lost:
        c.table[b, (n_rows[b] - 1) // page] = 10 ** 7
    want_k, want_v, want_w, bound_k = c.k_h.astype(np.float64), c.v_h.copy(), w.copy(), np.zeros(c.k_h.shape)
    kt, kb = treeref.turn(kn, pos, freq, rot, inter, 1.25)
    for b, n in enumerate(n_rows):
        at = pagedref.places(c.table_h, b, n, page)
        for i in range(q_len[b]):
            s, t = n - q_len[b] + i, q_start[b] + i
            want_w[b, :, s] = 0
            if b in lost and s // page == (n - 1) // page:
                continue
            want_k[at[s]], want_v[at[s]], bound_k[at[s]] = kt[t], vn[t], kb[t]
    wd, qd, out = dev(gpu, w), dev(gpu, q), gpu.full(q.shape, float("nan"), device="cuda")
    zt.paged_append_at(qd, dev(gpu, kn), dev(gpu, vn), out, c.k, c.v, c.table, dev(gpu, pos), freq, q_start, n_rows, page, H, Hkv,
                       d, rot, inter, 1.25, wd)
    got = out.cpu().numpy()
    want_q, bound_q = treeref.turn(q, pos, freq, rot, inter, 1.25)
    assert np.all(np.abs(got[1:N] - want_q[1:N]) <= bound_q[1:N]) and np.all(np.isnan(got[:1])) and np.all(np.isnan(got[N:]))
    assert np.all(np.abs(c.k.cpu().numpy() - want_k) <= bound_k) and np.array_equal(c.v.cpu().numpy(), want_v)
    assert np.array_equal(wd.cpu().numpy(), want_w)
    # q in place, and no q.
    c2 = c.k.clone()
    zt.paged_append_at(qd, dev(gpu, kn), dev(gpu, vn), qd, c.k, c.v, c.table, dev(gpu, pos), freq, q_start, n_rows, page, H, Hkv,
                       d, rot, inter, 1.25)
    assert np.array_equal(qd.cpu().numpy()[1:N], got[1:N]) and np.array_equal(qd.cpu().numpy()[N:], q[N:])
    zt.paged_append_at(None, dev(gpu, kn), dev(gpu, vn), None, c.k, c.v, c.table, dev(gpu, pos), freq, q_start, n_rows, page, H, Hkv,
                       d, rot, inter, 1.25)
    assert gpu.equal(c.k, c2)


# ---- pages ------------------------------------------------------------------------------------


@pytest.mark.parametrize("Hkv,d", [(2, 32), (8, 128), (3, 50), (1, 256), (5, 34)])
@pytest.mark.parametrize("page", [1, 8, 64])
def test_keep(gpu, zt, Hkv, d, page):
    """Lines of trees, one longer than a thread's batch of rows, numbers that move nothing, a count past the new tokens,
    a page that is none of the pool's."""
    rng = np.random.default_rng([Hkv, d, page])
    n_rows, q_len = [40, 0, 7, 64, 129, 31, 500] + [20] * 70, [3, 0, 7, 0, 60, 31, 40] + [4] * 70
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    q_start = np.cumsum([2] + q_len)
    path = np.full(q_start[-1] + 1, 12345, np.int32)
    count = np.zeros(len(n_rows), np.int32)
    for b, n in enumerate(q_len):
        if n:
            m = int(rng.integers(0, n + 1)) if b != 4 else 37
            path[q_start[b]:q_start[b] + m] = np.sort(rng.choice(n, m, replace=False))
            count[b] = m
    path[q_start[6]:q_start[6] + 8] = [0, 5, 4, 39, 39, 40, -1, 3]  # two that may not come here, one twice
    count[2], count[6], count[7] = 99, 8, -4
    path[q_start[2]:q_start[3]] = [1, 2, 3, 4, 5, 6, 6]
    table = c.table_h.copy()
    if page == 8:
        c.table[5, 2], table[5, 2] = -1, -1
    want_k, want_v = c.k_h.copy(), c.v_h.copy()
    for b, n in enumerate(n_rows):
        row0 = n - q_len[b]
        for i in range(min(max(count[b], 0), q_len[b])):
            p = path[q_start[b] + i]
            if not i <= p < q_len[b]:
                continue
            of, to = (table[b, (row0 + x) // page] * page + (row0 + x) % page if table[b, (row0 + x) // page] >= 0 else -1 for x in (p, i))
            if of >= 0 and to >= 0:
                want_k[to], want_v[to] = want_k[of], want_v[of]
    zt.paged_keep(c.k, c.v, c.table, dev(gpu, path), dev(gpu, count), q_start, n_rows, page, Hkv, d)
    assert np.array_equal(c.k.cpu().numpy(), want_k) and np.array_equal(c.v.cpu().numpy(), want_v)


class Pool:
    """Device tables and counts beside treeref.Pages."""

    def __init__(self, gpu, zt, B, stride, n_pages, page):
        self.gpu, self.zt, self.page = gpu, zt, page
        self.ref = treeref.Pages(np.full((B, stride), -1, np.int32), np.zeros(n_pages, np.int32), page)
        self.load()

    def load(self):
        self.table, self.refs = dev(self.gpu, self.ref.table), dev(self.gpu, self.ref.refs)

    def same(self):
        assert np.array_equal(self.table.cpu().numpy(), self.ref.table) and np.array_equal(self.refs.cpu().numpy(), self.ref.refs)

    def fork(self, src, dst, n_rows, n_room):
        gpu, n = self.gpu, len(src)
        pairs, missing = gpu.full((n + 1, 2), 7, device="cuda", dtype=gpu.int32), gpu.full((2,), 7, device="cuda", dtype=gpu.int32)
        need = self.zt.paged_fork_workspace_bytes(n_rows, n_room, len(self.ref.refs), self.page)
        ws = gpu.full((need // 4 + 1,), -9, device="cuda", dtype=gpu.int32)
        self.zt.paged_fork(self.table, self.refs, pairs, missing, src, dst, n_rows, n_room, self.page, ws[:-1])
        want, short = self.ref.fork(src, dst, n_rows, n_room)
        got = pairs.cpu().numpy()
        assert missing.tolist() == [short, 7] and np.array_equal(got[:n], want) and np.all(got[n] == 7) and int(ws[-1]) == -9
        self.same()
        return pairs[:n], short

    def free(self, n_keep):
        self.zt.paged_free(self.table, self.refs, n_keep, self.page)
        self.ref.free(n_keep)
        self.same()

    def compact(self, most, in_place):
        gpu = self.gpu
        pairs, moved = gpu.full((most, 2), 7, device="cuda", dtype=gpu.int32), gpu.full((3,), 7, device="cuda", dtype=gpu.int32)
        t, r = (self.table, self.refs) if in_place else (gpu.full_like(self.table, 9), gpu.full_like(self.refs, 9))
        before = self.table.clone(), self.refs.clone()
        ws = gpu.full((self.zt.paged_compact_workspace_bytes(len(self.ref.refs)) // 4,), -9, device="cuda", dtype=gpu.int32)
        self.zt.paged_compact(self.table, self.refs, t, r, pairs, moved, ws)
        want, counts = self.ref.compact(most)
        assert np.array_equal(pairs.cpu().numpy(), want) and moved.tolist() == counts + [7]
        if not in_place:
            assert gpu.equal(before[0], self.table) and gpu.equal(before[1], self.refs)
        self.table, self.refs = t, r
        self.same()
        return pairs


@pytest.mark.parametrize("B,stride,n_pages,page,lacks", [(6, 8, 20, 4, True), (200, 70, 4200, 16, True), (70, 300, 5000, 1, True),
                                                         (3, 5, 8192, 1024, False), (150, 4, 4097, 8, False),
                                                         (100, 500, 16385, 1, True), (200, 350, 20011, 2, True), (90, 40, 16384, 8, False),
                                                         (300, 5, 900, 8, False), (8, 600, 4300000, 1, False)])
def test_pages_in_use(gpu, zt, B, stride, n_pages, page, lacks):
    """Forks, growth, cuts, frees and compactions at random: tables and counts as treeref has them, the counts those of the
    tables; also calls that lack pages, and page tables that have been cut back into a shared page."""
    rng = np.random.default_rng([B, stride])
    pool, rows, lacked = Pool(gpu, zt, B, stride, n_pages, page), np.zeros(B, int), 0
    most = stride * page
    for step in range(25):
        slots = rng.permutation(B)
        n = int(rng.integers(1, B + 1))
        src, dst, n_rows, n_room = [], [], [], []
        empty = [b for b in slots if rows[b] == 0]
        full = [b for b in slots if rows[b] > 0]
        froms = set()
        for _ in range(n):
            if full and empty and rng.random() < 0.5:
                a = full[int(rng.integers(len(full)))]
                if a in dst:
                    continue
                froms.add(a)
                b, r = empty.pop(), int(rng.integers(0, rows[a] + 1))
            else:
                todo = [b for b in slots if b not in dst and b not in froms]
                if not todo:
                    break
                a = b = todo[0]
                r = rows[a]
                if b in empty:
                    empty.remove(b)
            src.append(a), dst.append(b), n_rows.append(r)
            n_room.append(int(min(most, r + rng.integers(0, max(2, most // 3)))))
        if src:
            _, short = pool.fork(src, dst, n_rows, n_room)
            lacked += short > 0
            if not short:
                rows[dst] = n_room
        cut = np.where(rng.random(B) < 0.5, rows, np.where(rng.random(B) < 0.4, 0, (rows * rng.random(B)).astype(int)))
        pool.free([most if c == rows[b] and rng.random() < 0.5 else int(c) for b, c in enumerate(cut)])
        rows = cut
        assert np.array_equal(pool.ref.refs, pool.ref.counted())
        if step % 3 == 2:
            pool.compact(int(rng.integers(1, 10)) if step % 2 else n_pages, in_place=step % 4 < 2)
    assert (lacked > 0) == lacks


@pytest.mark.parametrize("B,stride,n_pages,most", [(40, 512, 1, 1), (64, 192, 16384, 16384), (1, 12289, 16384, 9000), (64, 1024, 16384, 500),
                                                   (3, 6660, 1000, 1000), (3, 6661, 1000, 999), (5, 7, 4096, 9000), (5, 7, 4097, 4097),
                                                   (5, 7, 4097, 4098), (2, 20000, 900, 70000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compaction_of_small_and_of_wide_tables(gpu, zt, B, stride, n_pages, most, in_place):
    """Tables and pairs on both sides of what one workgroup is given; two thirds of the pool in use, some pages by several
    entries, a call that leaves pages to move and one that finishes."""
    rng = np.random.default_rng([B, stride, n_pages])
    p = Pool(gpu, zt, B, stride, n_pages, 1)
    live = rng.permutation(n_pages)[:max(1, min(2 * n_pages // 3, B * stride // 2))]
    at = rng.permutation(B * stride)[:len(live) + len(live) // 3]
    p.ref.table.reshape(-1)[at] = np.concatenate([live, live])[:len(at)]
    p.ref.table[0, :3] = [n_pages, -5, 2 ** 31 - 1]
    p.ref.refs[:] = p.ref.counted()
    p.load()
    for few in (7, most):
        p.compact(min(few, most), in_place)
        assert np.array_equal(p.ref.refs, p.ref.counted())


@pytest.mark.parametrize("B,stride,n_pages,most,one", [(8, 128, 1000, 500, True), (64, 192, 1000, 500, True), (64, 1024, 1000, 500, False),
                                                       (64, 1024, 16384, 500, False), (8, 128, 16384, 100000, False)])
def test_who_compacts(gpu, zt, B, stride, n_pages, most, one):
    """A single workgroup keeps its numbers to itself, three launches hand theirs on in the workspace: wide tables, and lists of
    pairs far beyond a large pool, are not left to one."""
    table, refs = gpu.full((B, stride), -1, device="cuda", dtype=gpu.int32), gpu.zeros(n_pages, device="cuda", dtype=gpu.int32)
    pairs, moved = gpu.full((most, 2), 7, device="cuda", dtype=gpu.int32), gpu.full((2,), 7, device="cuda", dtype=gpu.int32)
    table[0, 0], refs[n_pages - 1] = n_pages - 1, 1
    ws = gpu.full((zt.paged_compact_workspace_bytes(n_pages) // 4,), -9, device="cuda", dtype=gpu.int32)
    zt.paged_compact(table, refs, table, refs, pairs, moved, ws)
    assert pairs[0].tolist() == [n_pages - 1, 0] and bool((pairs[1:] == -1).all()) and moved.tolist() == [1, 0]
    assert int(table[0, 0]) == 0 and int(refs[0]) == 1 and int(refs.sum()) == 1
    assert bool((ws == -9).all()) == one


def test_entries_that_name_no_page(gpu, zt):
    """Numbers outside the pool in a table: shared as they are, not counted, replaced where a sequence grows, dropped where it is
    freed; compaction leaves them."""
    p = Pool(gpu, zt, 4, 6, 12, 4)
    p.ref.table[0, :5] = [3, 10 ** 6, 5, -7, -(2 ** 31)]
    p.ref.refs[[3, 5, 11]] = 1
    p.ref.table[3, 2] = 11
    p.load()
    pairs, _ = p.fork([0, 0], [1, 2], [15, 6], [17, 6])
    assert pairs.tolist() == [[-7, 0], [10 ** 6, 2]]  # (of which zt_paged_copy passes over)
    p.compact(3, True)
    p.fork([0], [0], [5], [20])
    p.free([3, 100, 0, 0])


@pytest.mark.parametrize("n_pages", [4096, 8192, 16384, 16385, 20480])
def test_a_full_pool_and_an_empty_one(gpu, zt, n_pages):
    p = Pool(gpu, zt, 2, n_pages + 100, n_pages, 1)
    p.compact(5, False)
    assert p.fork([0], [0], [0], [n_pages])[1] == 0
    p.compact(5, False)
    assert p.fork([1], [1], [0], [1])[1] == 1
    p.free([n_pages // 2 + 4, 0])
    assert p.fork([0], [1], [100], [100 + n_pages // 2 - 4])[1] == 0
    p.free([0, n_pages + 100])
    p.compact(n_pages, True)


def test_the_widest_tables(gpu, zt):
    """Tables of 2^31 - 1 columns, the most that an int counts: a fork, a compaction and a free reach their last column and
    leave what lies behind it."""
    stride, behind = 2 ** 31 - 1, 4096
    flat = gpu.full((2 * stride + behind,), 7, device="cuda", dtype=gpu.int32)
    flat[:stride] = -1
    table = flat[:2 * stride].view(2, stride)
    flat[0], flat[1] = 3, 5
    refs = gpu.tensor([0, 0, 0, 1, 0, 1, 1, 0], device="cuda", dtype=gpu.int32)
    pairs, missing = gpu.full((1, 2), 9, device="cuda", dtype=gpu.int32), gpu.full((1,), 9, device="cuda", dtype=gpu.int32)

    def holds(row0, row1):
        """The rows begin so; all else in the tables is -1, behind them 7."""
        for at, x in ((0, row0), (stride, row1)):
            assert flat[at:at + len(x)].tolist() == x
            for i in range(at + len(x), at + stride, 1 << 28):
                assert bool((flat[i:min(i + (1 << 28), at + stride)] == -1).all()), i
        assert bool((flat[2 * stride:] == 7).all())

    ws = gpu.empty(zt.paged_fork_workspace_bytes([6], [9], 8, 4), device="cuda", dtype=gpu.uint8)
    zt.paged_fork(table, refs, pairs, missing, [0], [1], [6], [9], 4, ws)
    assert pairs.tolist() == [[5, 0]] and missing.tolist() == [0] and refs.tolist() == [1, 1, 0, 2, 0, 1, 1, 0]
    holds([3, 5], [3, 0, 1])
    flat[stride - 1] = 6  # the last column's page moves, and is given back
    pairs, moved = gpu.full((8, 2), 9, device="cuda", dtype=gpu.int32), gpu.full((2,), 9, device="cuda", dtype=gpu.int32)
    ws = gpu.empty(zt.paged_compact_workspace_bytes(8), device="cuda", dtype=gpu.uint8)
    zt.paged_compact(table, refs, table, refs, pairs, moved, ws)
    assert pairs.tolist() == [[6, 2], [5, 4]] + [[-1, -1]] * 6 and moved.tolist() == [2, 0]
    assert int(flat[stride - 1]) == 2 and refs.tolist() == [1, 1, 1, 2, 1, 0, 0, 0]
    zt.paged_free(table, refs, [8, 4], 4)
    assert refs.tolist() == [0, 0, 0, 2, 1, 0, 0, 0]
    holds([3, 4], [3])


@pytest.mark.parametrize("page,Hkv,d", [(1, 2, 32), (8, 8, 128), (16, 3, 50), (64, 1, 34), (1024, 2, 256)])
def test_copy(gpu, zt, page, Hkv, d):
    rng = np.random.default_rng([page, d])
    n_pages = 12
    k, v = (rng.standard_normal((n_pages * page, Hkv, d)).astype(np.float32) for _ in range(2))
    pairs = [[3, 7], [-1, -1], [0, 1], [0, 11], [5, -1], [n_pages, 2], [2, n_pages], [10 ** 9, -(2 ** 31)]]
    kd, vd = dev(gpu, k), dev(gpu, v)
    zt.paged_copy(kd, vd, gpu.tensor(pairs, device="cuda", dtype=gpu.int32), page, Hkv, d)
    for x in (k, v):
        y = x.reshape(n_pages, -1)
        for of, to in ((3, 7), (0, 1), (0, 11)):
            y[to] = y[of]
    assert np.array_equal(kd.cpu().numpy(), k) and np.array_equal(vd.cpu().numpy(), v)


def test_more_copies_than_a_grid(gpu, zt):
    """600000 pairs, of which the last and a few others name pages."""
    k, v = gpu.randn(64, 4, 32, device="cuda"), gpu.randn(64, 4, 32, device="cuda")
    want = k.clone(), v.clone()
    pairs = np.full((600000, 2), -1, np.int32)
    for i, (of, to) in {0: (1, 2), 524287: (3, 4), 524288: (5, 6), 599999: (63, 0)}.items():
        pairs[i] = of, to
        for x in want:
            x[to] = x[of]
    zt.paged_copy(k, v, dev(gpu, pairs), 4, 1, 32)
    assert gpu.equal(k, want[0]) and gpu.equal(v, want[1])


def test_a_pool_past_32_bits(gpu, zt):
    """2^31 values and more in K and in V: appends, attention, moves and copies at its end as at its beginning."""
    H, Hkv, d, page, n, L = 8, 8, 128, 64, 150, 20
    n_pages = (1 << 31) // (page * Hkv * d) + 40
    rng = np.random.default_rng(3)
    k, v = (gpu.empty(n_pages, page, Hkv * d, device="cuda") for _ in range(2))
    head = gpu.randn(2, 3, page, Hkv * d, device="cuda")
    table = gpu.tensor([[0, 1, 2], [n_pages - 5, n_pages - 3, n_pages - 1]], device="cuda", dtype=gpu.int32)
    for b in range(2):
        k[table[b].long()], v[table[b].long()] = head[0], head[1]
    up = treeref.random_tree(rng, L)
    parent = dev(gpu, np.tile(up, 2))
    q_start, n_rows = [0, L, 2 * L], [n, n]
    mask, pos = gpu.empty(2 * L, 1, device="cuda", dtype=gpu.int64), gpu.empty(2 * L, device="cuda", dtype=gpu.int32)
    zt.tree_mask(parent, mask, q_start, pos, [n - L] * 2)
    new = [gpu.randn(L, Hkv * d, device="cuda").repeat(2, 1) for _ in range(3)]
    out = gpu.empty(2 * L, H * d, device="cuda")
    zt.paged_append_at(new[0], new[1], new[2], new[0], k, v, table, pos, zt.rope_frequencies(d), q_start, n_rows, page, H, Hkv, d, d)
    ws = gpu.empty(zt.attn_paged_workspace_bytes(q_start, n_rows, H, Hkv, d) + 16, device="cuda", dtype=gpu.uint8)
    zt.attn_paged_tree(new[0], k, v, table, mask, out, q_start, n_rows, page, H, Hkv, d, ws)
    line = max(treeref.lines(up), key=len)
    path = np.zeros(2 * L, np.int32)
    path[:len(line)] = path[L:L + len(line)] = line
    zt.paged_keep(k, v, table, dev(gpu, path), dev(gpu, np.full(2, len(line), np.int32)), q_start, n_rows, page, Hkv, d)
    assert gpu.equal(out[:L], out[L:]) and not bool(out.isnan().any())
    for x in (k, v):
        assert gpu.equal(x[table[0].long()], x[table[1].long()])
    zt.paged_copy(k, v, gpu.tensor([[n_pages - 5, n_pages - 20], [0, n_pages - 7]], device="cuda", dtype=gpu.int32), page, Hkv, d)
    for x in (k, v):
        assert gpu.equal(x[n_pages - 20], x[0]) and gpu.equal(x[n_pages - 7], x[0])


# ---- together -----------------------------------------------------------------------------------


def test_streams_and_graphs(gpu, zt):
    """Two streams at once, each with a workspace of its own, beside other work; then a graph of a step's calls, replayed
    with the program's own work between the replays, every replay checked."""
    H, Hkv, d, page, n_rows, q_len = 8, 2, 64, 16, [900, 300, 77], [26, 7, 40]
    rng = np.random.default_rng(8)
    q_start = np.cumsum([0] + list(q_len)).tolist()
    N = q_start[-1]
    parents = [treeref.random_tree(rng, n) for n in q_len]
    parent, (mask, depth) = dev(gpu, np.concatenate(parents)), treeref.masks(parents, 1)
    q = rng.standard_normal((N, H, d)).astype(np.float32)
    caches = [Cache(gpu, rng, n_rows, page, Hkv, d) for _ in range(2)]
    streams = [gpu.cuda.Stream() for _ in range(2)]
    outs = [gpu.empty(N, H, d, device="cuda") for _ in range(2)]
    wss = [gpu.empty(zt.attn_paged_workspace_bytes(q_start, n_rows, H, Hkv, d), device="cuda", dtype=gpu.uint8) for _ in range(2)]
    qd, md = dev(gpu, q), dev(gpu, mask)
    refs = [reference(c, q, mask, q_start, H) for c in caches]
    gpu.cuda.synchronize()
    for _ in range(10):
        for s, c, o, ws in zip(streams, caches, outs, wss):
            zt.attn_paged_tree(qd, c.k, c.v, c.table, md, o, q_start, n_rows, page, H, Hkv, d, ws, stream=s)
    gpu.cuda.synchronize()
    for o, ref in zip(outs, refs):
        check((o.cpu().numpy(), None, None), ref, q_start)

    c = caches[0]
    kn, vn, qo, m2, pos = (gpu.empty(N, Hkv, d, device="cuda"), gpu.empty(N, Hkv, d, device="cuda"), gpu.empty_like(qd),
                           gpu.zeros_like(md), gpu.zeros(N, device="cuda", dtype=gpu.int32))
    freq = zt.rope_frequencies(d)
    path, count = dev(gpu, np.zeros(N, np.int32)), dev(gpu, np.ones(3, np.int32))
    lines = [max(treeref.lines(up), key=len) for up in parents]
    for b, line in enumerate(lines):
        path[q_start[b]:q_start[b] + len(line)] = gpu.tensor(line, dtype=gpu.int32)
        count[b] = len(line)

    def step():
        zt.tree_mask(parent, m2, q_start, pos, [n - l for n, l in zip(n_rows, q_len)])
        zt.paged_append_at(qd, kn, vn, qo, c.k, c.v, c.table, pos, freq, q_start, n_rows, page, H, Hkv, d, d)
        zt.attn_paged_tree(qo, c.k, c.v, c.table, m2, outs[0], q_start, n_rows, page, H, Hkv, d, wss[0])
        zt.paged_keep(c.k, c.v, c.table, path, count, q_start, n_rows, page, Hkv, d)

    kn.normal_(), vn.normal_()
    step()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        step()
    for i in range(4):
        kn.normal_(), vn.normal_(), qd.normal_()
        step()
        gpu.cuda.synchronize()
        want = [x.clone() for x in (outs[0], c.k, c.v, m2, pos)]
        outs[0].fill_(float("nan")), m2.zero_(), pos.zero_()
        graph.replay()
        gpu.cuda.synchronize()
        assert all(gpu.equal(x, y) for x, y in zip(want, (outs[0], c.k, c.v, m2, pos)))
    assert np.array_equal(m2.cpu().numpy().view(np.uint64), mask) and np.array_equal(
        pos.cpu().numpy(), np.concatenate([np.full(l, n - l) for n, l in zip(n_rows, q_len)]) + depth)


def test_page_calls_in_a_graph(gpu, zt):
    """A beam step (free, fork, copy) and a compaction, captured and replayed on one state."""
    B, stride, n_pages, page, Hkv, d = 12, 40, 300, 4, 2, 32
    p = Pool(gpu, zt, B, stride, n_pages, page)
    p.fork([0, 1, 2], [0, 1, 2], [0] * 3, [61, 90, 33])
    k, v = (gpu.randn(n_pages * page, Hkv, d, device="cuda") for _ in range(2))
    src, dst, rows = [0, 0, 0, 1, 1, 2], [3, 4, 5, 6, 7, 2], [61, 61, 60, 90, 7, 33]
    room = [r + 9 for r in rows]
    pairs, missing = (gpu.empty(*s, device="cuda", dtype=gpu.int32) for s in ((6, 2), (1,)))
    ws = gpu.empty(zt.paged_fork_workspace_bytes(rows, room, n_pages, page), device="cuda", dtype=gpu.uint8)
    keep = [61, 90, 33] + [0] * 9
    cp, moved = gpu.empty(50, 2, device="cuda", dtype=gpu.int32), gpu.empty(2, device="cuda", dtype=gpu.int32)
    ws2 = gpu.empty(zt.paged_compact_workspace_bytes(n_pages), device="cuda", dtype=gpu.uint8)
    t2, r2 = gpu.empty_like(p.table), gpu.empty_like(p.refs)

    def step():
        zt.paged_free(p.table, p.refs, keep, page)
        zt.paged_fork(p.table, p.refs, pairs, missing, src, dst, rows, room, page, ws)
        zt.paged_copy(k, v, pairs, page, Hkv, d)
        zt.paged_compact(p.table, p.refs, t2, r2, cp, moved, ws2)

    step()
    gpu.cuda.synchronize()
    want = [x.clone() for x in (p.table, p.refs, pairs, missing, k, v, t2, r2, cp, moved)]
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        step()
    for i in range(4):
        for x in (pairs, missing, t2, r2, cp, moved):
            x.fill_(i)
        graph.replay()
        gpu.cuda.synchronize()
        assert all(gpu.equal(x, y) for x, y in zip(want, (p.table, p.refs, pairs, missing, k, v, t2, r2, cp, moved)))


@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 64), (6, 3, 50), (32, 8, 128)])
def test_weights_beside_trees(gpu, zt, H, Hkv, d):
    """A tree's step accumulates no weights: its rows have 0, the others keep theirs.  The accepted tokens attended once more, as
    a chunk, add what they draw, those rows among them."""
    n_rows, q_len, page, rot = [60, 200, 33, 9], [9, 40, 5, 9], 8, 24
    rng = np.random.default_rng([H, d, 5])
    c, B = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan), len(n_rows)
    q_start = np.cumsum([0] + q_len).tolist()
    N = q_start[-1]
    parents = [treeref.random_tree(rng, n, 0.8) for n in q_len]
    mask, pos = gpu.empty(N, 1, device="cuda", dtype=gpu.int64), gpu.empty(N, device="cuda", dtype=gpu.int32)
    zt.tree_mask(dev(gpu, np.concatenate(parents)), mask, q_start, pos, [n - L for n, L in zip(n_rows, q_len)])
    q, kn, vn = (dev(gpu, rng.standard_normal((N, h, d)).astype(np.float32)) for h in (H, Hkv, Hkv))
    w = rng.random((B, Hkv, max(n_rows) + 3), np.float32)
    wd, out = dev(gpu, w), gpu.empty(N, H, d, device="cuda")
    zt.paged_append_at(q, kn, vn, q, c.k, c.v, c.table, pos, zt.rope_frequencies(rot), q_start, n_rows, page, H, Hkv, d, rot, w=wd)
    ws = gpu.empty(zt.attn_paged_workspace_bytes(q_start, n_rows, H, Hkv, d) + 16, device="cuda", dtype=gpu.uint8)
    zt.attn_paged_tree(q, c.k, c.v, c.table, mask, out, q_start, n_rows, page, H, Hkv, d, ws)
    lines = [max(treeref.lines(up), key=len) for up in parents]
    path, count = np.zeros(N, np.int32), np.array([len(x) for x in lines], np.int32)
    for t0, line in zip(q_start, lines):
        path[t0:t0 + len(line)] = line
    zt.paged_keep(c.k, c.v, c.table, dev(gpu, path), dev(gpu, count), q_start, n_rows, page, Hkv, d)
    for b, (n, L) in enumerate(zip(n_rows, q_len)):
        w[b, :, n - L:n] = 0
    assert np.array_equal(wd.cpu().numpy(), w)
    rows = [n - L + len(x) for n, L, x in zip(n_rows, q_len, lines)]
    begin = np.cumsum([0] + [len(x) for x in lines]).tolist()
    took = np.concatenate([t0 + np.array(line) for t0, line in zip(q_start, lines)])
    q2 = q[dev(gpu, took)].contiguous()
    out2 = gpu.empty_like(q2)
    ws = gpu.empty(zt.attn_paged_workspace_bytes(begin, rows, H, Hkv, d, True), device="cuda", dtype=gpu.uint8)
    zt.attn_paged(q2, c.k, c.v, c.table, out2, begin, rows, page, H, Hkv, d, ws, w_in=wd, w_out=wd)
    k, v, got = c.k.cpu().numpy(), c.v.cpu().numpy(), wd.cpu().numpy()
    ref, _, drawn, bound, w_bound = pagedref.attend(q2.cpu().numpy(), k, v, c.table_h, begin, rows, page, H, Hkv, d)
    assert np.all(np.abs(out2.cpu().numpy() - ref) <= bound)
    for b, n in enumerate(rows):
        want = w[b, :, :n] + drawn[b, :, :n]
        assert np.all(np.abs(got[b, :, :n] - want) <= w_bound[b, :, :n] + 2 * EPS * np.abs(want))
        assert np.array_equal(got[b, :, n:], w[b, :, n:])
        assert np.all(got[b, :, n - len(lines[b]):n] > 0)


@pytest.mark.parametrize("H,Hkv,d,rot,inter", [(8, 2, 64, 64, False), (6, 3, 50, 24, True), (32, 8, 128, 64, False)])
def test_drafting(gpu, zt, H, Hkv, d, rot, inter):
    """Sequences that share a prompt's pages answer by drafted trees: each step they get room, the tree goes into the cache and
    is attended, one of its lines stays, and the rest's pages are freed; now and then a sequence is forked or dropped and
    the pool compacted.  Each token's output against a dense softmax over its sequence's true history, kept apart."""
    page, stride, n_pages, B, most = 8, 40, 170, 5, 12
    rng = np.random.default_rng([H, d])
    p = Pool(gpu, zt, B, stride, n_pages, page)
    k, v = (gpu.full((n_pages * page, Hkv, d), float("nan"), device="cuda") for _ in range(2))
    freq = zt.rope_frequencies(rot, 1e4, zt.ZT_ROPE_BASE, 4.0)
    hist = [[] for _ in range(B)]  # of each sequence: (position, turned k, v), in 64 bits
    live = [True] + [False] * (B - 1)

    def fork(src, dst):
        rows = [len(hist[a]) for a in src]
        pairs, short = p.fork(src, dst, rows, [r + most if a == b else r for a, b, r in zip(src, dst, rows)])
        assert short == 0
        zt.paged_copy(k, v, pairs, page, Hkv, d)
        for a, b in zip(src, dst):
            hist[b] = list(hist[a])
            live[b] = True

    for step in range(14):
        if step == 1:
            fork([0, 0, 0], [1, 2, 3])
        if step in (5, 9):
            gone = 1 if step == 5 else 2
            live[gone], hist[gone] = False, []
            p.free([len(h) for h in hist])
            fork([3], [gone])
            fork([0], [4]) if step == 5 else None
        if step in (6, 10):
            zt.paged_copy(k, v, p.compact(n_pages, step == 6), page, Hkv, d)
        on = [b for b in range(B) if live[b]]
        fork(on, on)
        q_len = [0 if not live[b] else int(rng.integers(1, most + 1)) for b in range(B)]
        if step == 0:
            q_len[0] = most
        parents = [np.arange(-1, n - 1, dtype=np.int32) if step == 0 else treeref.random_tree(rng, n) for n in q_len]
        q_start = np.cumsum([0] + list(q_len)).tolist()
        n_rows = [len(h) + n for h, n in zip(hist, q_len)]
        N = q_start[-1]
        first = [len(h) for h in hist]
        mask, pos = gpu.empty(N, 1, device="cuda", dtype=gpu.int64), gpu.empty(N, device="cuda", dtype=gpu.int32)
        zt.tree_mask(dev(gpu, np.concatenate(parents)), mask, q_start, pos, first)
        q, kn, vn = (rng.standard_normal((N, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
        qo, out = gpu.empty(N, H, d, device="cuda"), gpu.empty(N, H, d, device="cuda")
        zt.paged_append_at(dev(gpu, q), dev(gpu, kn), dev(gpu, vn), qo, k, v, p.table, pos, freq, q_start, n_rows, page, H, Hkv, d, rot,
                           inter)
        need = zt.attn_paged_workspace_bytes(q_start, n_rows, H, Hkv, d)
        ws = gpu.empty(need, device="cuda", dtype=gpu.uint8) if need else None
        zt.attn_paged_tree(qo, k, v, p.table, mask, out, q_start, n_rows, page, H, Hkv, d, ws)
        got = out.cpu().numpy()
        path, count = np.zeros(N, np.int32), np.zeros(B, np.int32)
        for b in on:
            lines = treeref.lines(parents[b])
            t0 = q_start[b]
            at = np.array([first[b] + len(line) - 1 for line in lines])
            qt, kt = (treeref.turn(x[t0:t0 + len(lines)], at, freq, rot, inter)[0] for x in (q, kn))
            for t, line in enumerate(lines):
                kk = np.array([x for x, _ in hist[b]] + [kt[j] for j in line])
                vv = np.array([x for _, x in hist[b]] + [vn[t0 + j].astype(np.float64) for j in line])
                for h in range(H):
                    ks, vs = kk[:, h * Hkv // H], vv[:, h * Hkv // H]
                    s = ks @ qt[t, h] / np.sqrt(d)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    # As treeref.attend's bound, with q's and k's own roundings (EPS each) in the scores.
                    e = 2 * (d + 6) * EPS * (np.abs(ks) @ np.abs(qt[t, h])).max() / np.sqrt(d)
                    n = n_rows[b]
                    assert np.all(np.abs(got[t0 + t, h] - w @ vs) <= (np.expm1(e) + (n + n / 16 + 32) * EPS) * (w @ np.abs(vs)))
            line = lines[int(rng.integers(len(lines)))] if step else lines[-1]
            path[t0:t0 + len(line)], count[b] = line, len(line)
            hist[b] += [(kt[j], vn[t0 + j].astype(np.float64)) for j in line]
        zt.paged_keep(k, v, p.table, dev(gpu, path), dev(gpu, count), q_start, n_rows, page, Hkv, d)
        p.free([len(h) for h in hist])
        assert np.array_equal(p.ref.refs, p.ref.counted())
