"""The paged cache on the GPU against pagedref (64 bits): append, attention of one and more new tokens, accumulated
weights, eviction, and a serving run of all of them."""
import numpy as np
import pytest

import pagedref

pytestmark = pytest.mark.gpu
EPS = pagedref.EPS


class Cache:
    """Pools and tables of a ragged batch; pages dealt at random, entries behind a sequence's last name no page."""

    def __init__(self, torch, rng, n_rows, page, Hkv, d, spare=1, garbage=None):
        used = [-(-n // page) for n in n_rows]
        self.n_rows, self.page, self.Hkv, self.d = list(n_rows), page, Hkv, d
        self.n_pages = sum(used) + spare
        order = rng.permutation(self.n_pages)
        self.table_h = np.full((len(n_rows), max(max(used), 1)), -1, np.int32)
        at = 0
        for b, u in enumerate(used):
            self.table_h[b, :u] = order[at:at + u]
            at += u
        shape = (self.n_pages * page, Hkv, d)
        self.k_h, self.v_h = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
        if garbage is not None:  # rows that are nobody's
            mine = np.zeros(shape[0], bool)
            for b, n in enumerate(n_rows):
                mine[pagedref.places(self.table_h, b, n, page)] = True
            self.k_h[~mine] = garbage
            self.v_h[~mine] = garbage
        self.k, self.v, self.table = (torch.from_numpy(x.copy()).cuda() for x in (self.k_h, self.v_h, self.table_h))


def run_attend(gpu, zt, c, q_h, q_start, H, w_h=None, lse=True, stream=None):
    """out, lse, w as numpy; buffers' rows that no token has, and the workspace, begin as NaN."""
    q = gpu.from_numpy(np.ascontiguousarray(q_h, np.float32)).cuda()
    out = gpu.full_like(q, float("nan"))
    l = gpu.full(q.shape[:2], float("nan"), device="cuda") if lse else None
    w_in = None if w_h is None else gpu.from_numpy(w_h.copy()).cuda()
    w_out = None if w_h is None else gpu.full_like(w_in, -7.0)
    need = zt.attn_paged_workspace_bytes(q_start, c.n_rows, H, c.Hkv, c.d, w_h is not None)
    ws = gpu.full((need // 4,), float("nan"), device="cuda") if need else None
    if stream is not None:
        stream.wait_stream(gpu.cuda.current_stream())
    zt.attn_paged(q, c.k, c.v, c.table, out, q_start, c.n_rows, c.page, H, c.Hkv, c.d, ws, l, w_in, w_out, stream)
    gpu.cuda.synchronize()
    return [None if t is None else t.cpu().numpy() for t in (out, l, w_out)]


def grade(got, ref, q_start, n_rows, Hkv, w_h=None):
    out, lse, w = got
    r_out, r_lse, r_w, bound, w_bound = ref
    rows = slice(q_start[0], q_start[-1])
    assert np.all(np.abs(out[rows] - r_out[rows]) <= bound[rows])
    assert np.all(np.isnan(out[:q_start[0]])) and np.all(np.isnan(out[q_start[-1]:]))
    if lse is not None:
        # The scores' error, the sum's (at most expm1(e) + n EPS, in `bound`'s terms) and the logarithm's.
        top = (bound[rows] / np.maximum(np.abs(r_out[rows]), 1e-30)).min(-1)
        assert np.all(np.abs(lse[rows] - r_lse[rows]) <= top + 4 * EPS * np.abs(r_lse[rows]) + 8 * EPS)
        assert np.all(np.isnan(lse[:q_start[0]])) and np.all(np.isnan(lse[q_start[-1]:]))
    if w_h is not None:
        for b, n in enumerate(n_rows):
            want = w_h[b, :, :n] + r_w[b, :, :n]
            assert np.all(np.abs(w[b, :, :n] - want) <= w_bound[b, :, :n] + 2 * EPS * np.abs(want))
            assert np.all(w[b, :, n:] == -7.0)


SHAPES = [(4, 2, 32), (8, 8, 64), (6, 2, 64), (32, 8, 128), (8, 2, 96), (16, 4, 256), (5, 1, 128), (40, 2, 32), (2, 1, 160),
          (4, 4, 34), (6, 3, 50), (9, 3, 250), (8, 2, 132), (4, 1, 192), (8, 4, 40), (64, 1, 64), (33, 1, 32)]
# (rows with the new tokens, new tokens): one token, none, no rows, ends inside a 16-key tile and at it, prompts.
BATCHES = {
    "single_tokens": ([1, 2, 15, 16, 17, 33, 200], [1] * 7),
    "ragged": ([40, 0, 7, 64, 129, 31, 5], [3, 0, 7, 0, 17, 31, 1]),
    "long": ([700], [2]),
    "chunk": ([333], [90]),
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("page", [1, 8, 16, 64])
@pytest.mark.parametrize("H,Hkv,d", SHAPES)
def test_attention_and_weights(gpu, zt, H, Hkv, d, page, batch):
    n_rows, q_len = BATCHES[batch]
    rng = np.random.default_rng([H, Hkv, d, page, len(n_rows)])
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([2] + q_len).tolist()  # the packed tokens begin behind two that are not this call's
    q = rng.standard_normal((q_start[-1] + 3, H, d)).astype(np.float32)
    w = rng.random((len(n_rows), Hkv, max(n_rows) + 5), np.float32)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)
    plain = run_attend(gpu, zt, c, q, q_start, H, lse=False)
    grade(plain, ref, q_start, n_rows, Hkv)
    # In whole: the 2-norm of the difference, roundings adding up as independent ones, with a factor of four.
    rows, n = slice(q_start[0], q_start[-1]), max(n_rows)
    off = np.linalg.norm(plain[0][rows] - ref[0][rows]) / np.linalg.norm(ref[0][rows])
    assert off <= 4 * EPS * (np.sqrt(d) + np.sqrt(n) + 16)


@pytest.mark.parametrize("settings", [{"ZT_PAGED_SCORES": 0}, {"ZT_PAGED_SCORES": 1}, {"ZT_PAGED_WGS": 256},
                                      {"ZT_PAGED_WGS": 32768}])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 8, 64), (8, 2, 96), (32, 8, 128), (6, 2, 50), (4, 1, 192), (8, 2, 256),
                                     (3, 1, 250)])
def test_forced_variants(gpu, zt, tune, settings, H, Hkv, d):
    """Weights from kept scores and from scores formed again, and other splits of the keys."""
    n_rows, q_len, page = [600, 90, 1300, 333], [300, 9, 1, 41], 16
    rng = np.random.default_rng([H, d])
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([0] + q_len).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    w = rng.random((4, Hkv, max(n_rows) + 5), np.float32)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    tune(settings)
    grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)


@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 64), (6, 2, 50), (8, 2, 96), (32, 8, 128), (8, 2, 192), (16, 4, 256)])
def test_a_batch_and_its_sequences_alone(gpu, zt, H, Hkv, d):
    """Few and many new tokens in one call, whose short sequences share a launch, and each of them in a call of its own."""
    n_rows, q_len, page = [300, 77, 9, 140, 33, 1, 260], [1, 4, 8, 9, 33, 1, 130], 8
    rng = np.random.default_rng([H, d, 7])
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([1] + q_len).tolist()
    q = rng.standard_normal((q_start[-1] + 2, H, d)).astype(np.float32)
    w = rng.random((len(n_rows), Hkv, max(n_rows) + 5), np.float32)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)
    table = c.table
    for b, n in enumerate(n_rows):
        c.table, c.n_rows = table[b:b + 1].contiguous(), [n]
        mine = [x[b:b + 1] if i in (2, 4) else x for i, x in enumerate(ref)]
        grade(run_attend(gpu, zt, c, q, q_start[b:b + 2], H, w[b:b + 1]), mine, q_start[b:b + 2], [n], Hkv, w[b:b + 1])


def test_more_sequences_than_a_launch_takes(gpu, zt):
    B, H, Hkv, d, page = 150, 4, 2, 32, 8
    rng = np.random.default_rng(5)
    n_rows = [int(x) for x in rng.integers(0, 60, B)]
    n_rows[70] = 2500  # enough to be cut into chunks
    q_len = [min(n, int(rng.integers(0, 12)) if i % 3 else 1) for i, n in enumerate(n_rows)]
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.inf)
    q_start = np.cumsum([0] + q_len).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    w = rng.random((B, Hkv, max(n_rows)), np.float32)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("L,n", [(9, 40), (70, 130), (150, 150)])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 128), (6, 2, 50), (4, 1, 256)])
def test_what_a_token_does_not_see_changes_nothing(gpu, zt, H, Hkv, d, L, n, value):
    """K and V of the last token's row not finite: tokens before it as without, bit for bit; it itself as 64 bits have it."""
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [n], 16, Hkv, d)
    q = rng.standard_normal((L, H, d)).astype(np.float32)
    w = np.zeros((1, Hkv, n), np.float32)
    out0, lse0, w0 = run_attend(gpu, zt, c, q, [0, L], H, w)
    last = pagedref.places(c.table_h, 0, n, 16)[-1]
    c.v[last, :, 3] = float(value)
    out1, lse1, w1 = run_attend(gpu, zt, c, q, [0, L], H, w)
    assert np.array_equal(out0[:-1], out1[:-1]) and np.array_equal(lse0, lse1) and np.array_equal(w0, w1)
    keep = np.arange(d) != 3
    assert np.array_equal(out0[-1][:, keep], out1[-1][:, keep])
    assert np.all(np.isnan(out1[-1, :, 3]) if np.isnan(value) else out1[-1, :, 3] == value)
    c.k[last] = float(value)
    out2, lse2, w2 = run_attend(gpu, zt, c, q, [0, L], H, w)
    assert np.array_equal(out0[:-1], out2[:-1]) and np.array_equal(lse0[:-1], lse2[:-1])
    # inf * q over columns of both signs: NaN scores, and with them the token's whole row.
    assert np.all(np.isnan(out2[-1])) and np.all(np.isnan(lse2[-1]))


@pytest.mark.parametrize("scores", [0, 1])
@pytest.mark.parametrize("L", [5, 40, 150])
@pytest.mark.parametrize("where", ["k", "q", "both", "v"])
@pytest.mark.parametrize("H,Hkv,d", [(8, 2, 64), (8, 2, 128), (4, 1, 256), (6, 2, 50)])
def test_large_values(gpu, zt, tune, H, Hkv, d, where, L, scores):
    """Values past 2^40 (kept out of the split products and added from the full rows): in K against as small ones in Q,
    the other way round, both, and in V."""
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
    c.k, c.v = gpu.from_numpy(c.k_h).cuda(), gpu.from_numpy(c.v_h).cuda()
    w = rng.random((1, Hkv, n), np.float32)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, [0, L], [n], page, H, Hkv, d)
    tune({"ZT_PAGED_SCORES": scores})
    grade(run_attend(gpu, zt, c, q, [0, L], H, w), ref, [0, L], [n], Hkv, w)


def test_no_new_tokens(gpu, zt):
    """Weights are copied, nothing else happens; no tokens and no weights: nothing at all."""
    H, Hkv, d, page, n_rows = 4, 2, 32, 8, [30, 0, 2000]
    rng = np.random.default_rng(31)
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    w = rng.random((3, Hkv, 2001), np.float32)
    out, lse, got = run_attend(gpu, zt, c, np.zeros((2, H, d)), [1, 1, 1, 1], H, w)
    assert np.all(np.isnan(out)) and np.all(np.isnan(lse))
    for b, n in enumerate(n_rows):
        assert np.array_equal(got[b, :, :n], w[b, :, :n]) and np.all(got[b, :, n:] == -7.0)
    out, lse, _ = run_attend(gpu, zt, c, np.zeros((2, H, d)), [1, 1, 1, 1], H)
    assert np.all(np.isnan(out)) and np.all(np.isnan(lse))
    k, before = gpu.zeros(1, Hkv * d, device="cuda"), c.k.clone()
    zt.paged_append(None, k, k, None, c.k, c.v, c.table, [1, 1, 1, 1], n_rows, [0, 0, 0], page, H, Hkv, d)
    assert gpu.equal(c.k, before)


def test_the_binding_checks_what_the_library_cannot_see(gpu, zt):
    H, Hkv, d, page = 4, 2, 32, 8
    c = Cache(gpu, np.random.default_rng(32), [30], page, Hkv, d)
    q, w = gpu.zeros(3, H * d, device="cuda"), gpu.zeros(1, Hkv, 30, device="cuda")
    kept = gpu.empty(1, Hkv, 8, device="cuda", dtype=gpu.int32)
    for bad in (dict(q=q[:2].contiguous()), dict(out=q[:2].contiguous()), dict(w_in=w, w_out=w[:, :1].contiguous()),
                dict(v=c.v[:-1].contiguous()), dict(table=c.table.long()), dict(q_start=[0, 1, 3])):
        a = dict(q=q, out=gpu.empty_like(q), v=c.v, table=c.table, q_start=[0, 3], w_in=None, w_out=None)
        a.update(bad)
        with pytest.raises(ValueError):
            zt.attn_paged(a["q"], c.k, a["v"], a["table"], a["out"], a["q_start"], [30], page, H, Hkv, d, None, None,
                          a["w_in"], a["w_out"])
    with pytest.raises(zt.ZtRefused):  # a null w_in beside a w_out
        zt.attn_paged(q, c.k, c.v, c.table, gpu.empty_like(q), [0, 3], [30], page, H, Hkv, d, None, None, None, w)
    with pytest.raises(ValueError):
        zt.paged_append(None, q, q, None, c.k, c.v, c.table, [0, 30], [30], [0], page, H, Hkv, d)
    with pytest.raises(ValueError):
        zt.paged_evict(c.k, c.v, c.table, c.table, w, w, kept, [30], page, Hkv, d, 1, 1, 9)


def test_sequences_that_share_pages(gpu, zt):
    """Three sequences over one prefix, the third the first again."""
    H, Hkv, d, page = 8, 2, 64, 16
    rng = np.random.default_rng(21)
    n_rows, q_len = [100, 90, 100], [3, 40, 3]
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    c.table_h[1, :5] = c.table_h[0, :5]
    c.table_h[2] = c.table_h[0]
    c.table = gpu.from_numpy(c.table_h).cuda()
    q_start = np.cumsum([0] + q_len).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    q[-3:] = q[:3]
    w = np.repeat(rng.random((1, Hkv, 100), np.float32), 3, 0)
    ref = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    got = run_attend(gpu, zt, c, q, q_start, H, w)
    grade(got, ref, q_start, n_rows, Hkv, w)
    assert np.array_equal(got[0][:3], got[0][-3:]) and np.array_equal(got[2][0], got[2][2])


@pytest.mark.parametrize("bad", [-1, 10 ** 9, "n_pages"])
@pytest.mark.parametrize("L", [6, 80])
def test_a_page_of_no_pool_is_not_followed(gpu, zt, bad, L):
    H, Hkv, d, page, n = 4, 2, 64, 8, 200
    rng = np.random.default_rng(9)
    c = Cache(gpu, rng, [n, n], page, Hkv, d)
    q = rng.standard_normal((2 * L, H, d)).astype(np.float32)
    q_start, w = [0, L, 2 * L], np.zeros((2, Hkv, n), np.float32)
    good = run_attend(gpu, zt, c, q, q_start, H, w)
    c.table[1, -1] = c.n_pages if bad == "n_pages" else bad  # sequence 1's last 8 rows
    out, lse, w1 = run_attend(gpu, zt, c, q, q_start, H, w)
    see = 2 * L - min(L, page)  # the first token that sees one of them
    assert np.array_equal(out[:see], good[0][:see]) and np.array_equal(lse[:see], good[1][:see])
    assert np.all(np.isnan(out[see:])) and np.all(np.isnan(lse[see:]))
    assert np.array_equal(w1[0], good[2][0]) and np.all(np.isnan(w1[1]))


@pytest.mark.parametrize("H,Hkv,d,page", [(4, 2, 32, 1), (32, 8, 128, 16), (6, 2, 50, 8), (16, 4, 256, 64), (3, 1, 34, 4)])
@pytest.mark.parametrize("with_q", [True, False])
def test_append(gpu, zt, H, Hkv, d, page, with_q):
    rng = np.random.default_rng([H, d])
    n_rows = [int(x) for x in rng.integers(0, 90, 80)]
    q_len = [min(n, [0, 1, 3, 40][i % 4]) for i, n in enumerate(n_rows)]
    pos = [n - l + 5000 * (i % 2) for i, (n, l) in enumerate(zip(n_rows, q_len))]
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    q_start = np.cumsum([3] + q_len).tolist()
    N = q_start[-1] + 2
    q, kn, vn = (rng.standard_normal((N, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
    w = rng.random((80, Hkv, max(n_rows) + 1), np.float32)
    dq, dk, dv, dw = (gpu.from_numpy(x).cuda() for x in (q, kn, vn, w))
    q_out = gpu.full_like(dq, -7.0)
    zt.paged_append(dq if with_q else None, dk, dv, q_out if with_q else None, c.k, c.v, c.table, q_start, n_rows, pos, page,
                    H, Hkv, d, 10000.0, dw)
    gpu.cuda.synchronize()
    k, v, q_want = c.k_h.astype(np.float64), c.v_h.copy(), np.full(q.shape, -7.0)
    for b, n in enumerate(n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        at = pagedref.places(c.table_h, b, n, page)[n - (t1 - t0):]
        k[at], v[at] = pagedref.rotate(kn[t0:t1], pos[b], 10000.0), vn[t0:t1]
        q_want[t0:t1] = pagedref.rotate(q[t0:t1], pos[b], 10000.0)
        w[b, :, n - (t1 - t0):n] = 0
    # One rounding to f32 of a value in 64 bits: half a step, and the 64-bit angle's own error (5000 radians x 2^-52).
    assert np.all(np.abs(c.k.cpu().numpy() - k) <= EPS * np.abs(k) + 1e-11)
    assert np.array_equal(c.v.cpu().numpy(), v) and np.array_equal(dw.cpu().numpy(), w)
    if with_q:
        assert np.all(np.abs(q_out.cpu().numpy() - q_want) <= EPS * np.abs(q_want) + 1e-11)
        zt.paged_append(dq, dk, dv, dq, c.k, c.v, c.table, q_start, n_rows, pos, page, H, Hkv, d, 10000.0)  # in place
        rows = slice(q_start[0], q_start[-1])
        assert gpu.equal(dq[rows], q_out[rows])


def test_append_rotates_as_the_contiguous_entry_does(gpu, zt):
    """Bit for bit what zt_rope_qk_forward writes."""
    T, H, Hkv, d = 37, 8, 2, 64
    rng = np.random.default_rng(2)
    c = Cache(gpu, rng, [T], 16, Hkv, d)
    q, k, v = (gpu.randn(T, h, d, device="cuda") for h in (H, Hkv, Hkv))
    q_out, q_rope, k_rope = gpu.empty_like(q), gpu.empty_like(q), gpu.empty_like(k)
    zt.paged_append(q, k, v, q_out, c.k, c.v, c.table, [0, T], [T], [11], 16, H, Hkv, d)
    zt.rope_qk(q, k, q_rope, k_rope, 1, T, H, Hkv, d, pos=11)
    at = gpu.from_numpy(pagedref.places(c.table_h, 0, T, 16)).cuda()
    assert gpu.equal(q_out, q_rope) and gpu.equal(c.k[at], k_rope)


def test_append_writes_no_page_of_no_pool(gpu, zt):
    H, Hkv, d, page = 2, 2, 32, 4
    rng = np.random.default_rng(4)
    c = Cache(gpu, rng, [12], page, Hkv, d, spare=3)
    c.table[0, 1], c.table[0, 2] = -5, c.n_pages
    before = c.k.clone(), c.v.clone()
    k, v = gpu.randn(12, Hkv, d, device="cuda"), gpu.randn(12, Hkv, d, device="cuda")
    zt.paged_append(None, k, v, None, c.k, c.v, c.table, [0, 12], [12], [0], page, H, Hkv, d)
    first = gpu.from_numpy(pagedref.places(c.table_h, 0, 4, page)).cuda()
    assert gpu.equal(c.v[first], v[:4])
    before[0][first], before[1][first] = c.k[first], c.v[first]
    assert gpu.equal(c.k, before[0]) and gpu.equal(c.v, before[1])


def _weights(rng, B, Hkv, n, kind):
    w = rng.random((B, Hkv, n), np.float32) ** 4 * 8
    if kind == "ties":
        w = np.floor(w)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "odd":  # everything that f32 holds
        w = rng.integers(0, 1 << 32, (B, Hkv, n), dtype=np.uint32).view(np.float32).copy()
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -0.0
        w[rng.random(w.shape) < 0.1] = 0.0
    return w


@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_rows,budget,first,last,Hkv,d,page", [
    ([40, 7, 33, 0, 32], 32, 4, 8, 2, 32, 1), ([500, 130, 129], 128, 0, 0, 8, 128, 16), ([200, 90], 64, 32, 32, 3, 50, 8),
    ([2100], 1, 0, 0, 1, 64, 16), ([2100], 1, 1, 0, 2, 34, 16), ([5000, 1500], 1300, 4, 64, 2, 96, 64),
    ([300], 299, 0, 7, 4, 256, 4), ([90, 20], 200, 4, 4, 2, 32, 8), ([20000], 9000, 1, 1, 1, 32, 16)])
def test_eviction(gpu, zt, n_rows, budget, first, last, Hkv, d, page, in_place, kind):
    rng = np.random.default_rng([len(n_rows), budget, d])
    B, stride = len(n_rows), max(n_rows) + 3
    c = Cache(gpu, rng, n_rows + [budget] * B, page, Hkv, d)
    table = c.table[:B].contiguous()
    table_out = table if in_place else c.table[B:].contiguous()
    out_h = c.table_h[:B] if in_place else c.table_h[B:]
    w = _weights(rng, B, Hkv, stride, kind)
    w_in = gpu.from_numpy(w).cuda()
    w_out = w_in if in_place else gpu.full_like(w_in, -7.0)
    kept = gpu.full((B, Hkv, budget), 12345, device="cuda", dtype=gpu.int32)
    zt.paged_evict(c.k, c.v, table, table_out, w_in, w_out, kept, n_rows, page, Hkv, d, first, last, budget)
    gpu.cuda.synchronize()
    k, v = c.k_h.copy(), c.v_h.copy()
    w_want = w.copy() if in_place else np.full_like(w, -7.0)
    kept_want = np.full((B, Hkv, budget), -1)
    for b, n in enumerate(n_rows):
        src = pagedref.places(c.table_h, b, n, page)
        dst = pagedref.places(out_h, b, min(n, budget), page)
        for h in range(Hkv):
            rows = pagedref.evict(w[b, h], n, budget, first, last)
            kept_want[b, h, :len(rows)] = rows
            k[dst, h], v[dst, h] = c.k_h[src[rows], h], c.v_h[src[rows], h]
            w_want[b, h, :len(rows)] = w[b, h, rows]
    assert np.array_equal(kept.cpu().numpy(), kept_want)
    assert np.array_equal(c.k.cpu().numpy(), k) and np.array_equal(c.v.cpu().numpy(), v)
    assert np.array_equal(w_out.cpu().numpy().view(np.uint32), w_want.view(np.uint32))


def test_eviction_of_many_sequences(gpu, zt):
    B, Hkv, d, page, budget = 130, 2, 32, 8, 24
    rng = np.random.default_rng(6)
    n_rows = [int(x) for x in rng.integers(0, 60, B)]
    c = Cache(gpu, rng, n_rows, page, Hkv, d)
    w = rng.random((B, Hkv, 60), np.float32)
    w_dev = gpu.from_numpy(w).cuda()
    kept = gpu.empty((B, Hkv, budget), device="cuda", dtype=gpu.int32)
    zt.paged_evict(c.k, c.v, c.table, c.table, w_dev, w_dev, kept, n_rows, page, Hkv, d, 2, 5, budget)
    kept, k = kept.cpu().numpy(), c.k.cpu().numpy()
    for b, n in enumerate(n_rows):
        at = pagedref.places(c.table_h, b, n, page)
        for h in range(Hkv):
            rows = pagedref.evict(w[b, h], n, budget, 2, 5)
            assert np.array_equal(kept[b, h, :len(rows)], rows) and np.all(kept[b, h, len(rows):] == -1)
            assert np.array_equal(k[at[:len(rows)], h], c.k_h[at[rows], h])


def test_eviction_follows_no_page_of_no_pool(gpu, zt):
    Hkv, d, page, budget = 2, 32, 4, 8
    rng = np.random.default_rng(8)
    for in_place in (True, False):
        c = Cache(gpu, rng, [20, 8], page, Hkv, d)
        w = gpu.rand(1, Hkv, 20, device="cuda")
        table = c.table[:1].clone()
        table[0, 3] = c.n_pages + 7
        out = table if in_place else c.table[1:].clone()
        kept = gpu.empty((1, Hkv, budget), device="cuda", dtype=gpu.int32)
        zt.paged_evict(c.k, c.v, table, out, w, w.clone() if not in_place else w, kept, [20], page, Hkv, d, 1, 2, budget)
        rows = kept.cpu().numpy()[0]
        src = pagedref.places(c.table_h, 0, 20, page)
        dst = src[:budget] if in_place else pagedref.places(c.table_h, 1, budget, page)
        want = c.k_h.copy()
        for h in range(Hkv):
            ok = rows[h] // page != 3  # rows of the page that is none stay where they were
            want[dst[ok], h] = c.k_h[src[rows[h][ok]], h]
        assert np.array_equal(c.k.cpu().numpy(), want)


def test_offsets_past_32_bits(gpu, zt):
    """A pool of 4.3e9 floats: rows whose element offsets do not fit 32 bits."""
    H, Hkv, d, page, n = 8, 8, 256, 64, 200
    pool_rows = (1 << 32) // (Hkv * d) // page * page + 4 * page
    rng = np.random.default_rng(12)
    c = Cache(gpu, rng, [n], page, Hkv, d, spare=0)
    k, v = (gpu.empty(pool_rows * Hkv * d, device="cuda") for _ in range(2))
    far = pool_rows // page - c.n_pages  # the pool's last pages take the small pool's place
    k[far * page * Hkv * d:], v[far * page * Hkv * d:] = c.k.view(-1), c.v.view(-1)
    near = c.k, c.v, c.table
    q = rng.standard_normal((3, H, d)).astype(np.float32)
    w = rng.random((1, Hkv, n), np.float32)
    want = run_attend(gpu, zt, c, q, [0, 3], H, w)
    many = rng.standard_normal((150, H, d)).astype(np.float32)
    want_many = run_attend(gpu, zt, c, many, [0, 150], H, w)
    c.k, c.v, c.table = k, v, near[2] + far
    got = run_attend(gpu, zt, c, q, [0, 3], H, w)
    got_many = run_attend(gpu, zt, c, many, [0, 150], H, w)
    for x, y in zip(want + want_many, got + got_many):
        assert np.array_equal(x, y)
    new = gpu.randn(2, Hkv * d, device="cuda")
    for kk, vv, table in (near, (k, v, c.table)):
        zt.paged_append(None, new, new, None, kk, vv, table, [0, 2], [n], [n - 2], page, H, Hkv, d)
    kept = gpu.empty((1, Hkv, 50), device="cuda", dtype=gpu.int32)
    for kk, vv, table in (near, (k, v, c.table)):
        wd = gpu.from_numpy(w).cuda()
        zt.paged_evict(kk, vv, table, table, wd, wd, kept, [n], page, Hkv, d, 1, 3, 50)
    assert gpu.equal(k[far * page * Hkv * d:], near[0].view(-1)) and gpu.equal(v[far * page * Hkv * d:], near[1].view(-1))


def test_other_streams_and_two_at_once(gpu, zt):
    H, Hkv, d, page = 8, 2, 64, 16
    rng = np.random.default_rng(14)
    cs = [Cache(gpu, rng, [900, 300], page, Hkv, d) for _ in range(2)]
    q = rng.standard_normal((5, H, d)).astype(np.float32)
    w = rng.random((2, Hkv, 900), np.float32)
    want = [run_attend(gpu, zt, c, q, [0, 1, 5], H, w) for c in cs]
    streams = [gpu.cuda.Stream() for _ in range(2)]
    got = [run_attend(gpu, zt, c, q, [0, 1, 5], H, w, stream=s) for c, s in zip(cs, streams)]
    for x, y in zip(sum(want, []), sum(got, [])):
        assert np.array_equal(x, y)
    # Both in flight together, each with its own buffers.
    dq = gpu.from_numpy(q).cuda()
    need = zt.attn_paged_workspace_bytes([0, 1, 5], [900, 300], H, Hkv, d)
    outs = [gpu.empty_like(dq) for _ in cs]
    spaces = [gpu.empty(need + 16, device="cuda", dtype=gpu.uint8) for _ in cs]
    gpu.cuda.synchronize()
    for _ in range(20):
        for c, s, o, ws in zip(cs, streams, outs, spaces):
            zt.attn_paged(dq, c.k, c.v, c.table, o, [0, 1, 5], [900, 300], page, H, Hkv, d, ws, stream=s)
    gpu.cuda.synchronize()
    for o, x in zip(outs, want):
        assert np.array_equal(o.cpu().numpy(), x[0])


def test_two_graphs_with_one_workspace(gpu, zt):
    """Two captured calls of different lengths that share a workspace, replayed in turn on one stream."""
    H, Hkv, d, page = 8, 2, 64, 16
    rng = np.random.default_rng(16)
    cs = [Cache(gpu, rng, n, page, Hkv, d) for n in ([1500, 700], [300])]
    starts = [[0, 1, 41], [0, 90]]
    qs = [gpu.from_numpy(rng.standard_normal((s[-1], H, d)).astype(np.float32)).cuda() for s in starts]
    ws_w = [gpu.from_numpy(rng.random((len(c.n_rows), Hkv, max(c.n_rows)), np.float32)).cuda() for c in cs]
    need = max(zt.attn_paged_workspace_bytes(s, c.n_rows, H, Hkv, d, True) for s, c in zip(starts, cs))
    ws = gpu.empty(need, device="cuda", dtype=gpu.uint8)
    outs, w_outs = [gpu.zeros_like(q) for q in qs], [gpu.zeros_like(w) for w in ws_w]  # (later w_out: left as it is)

    def call(i):
        zt.attn_paged(qs[i], cs[i].k, cs[i].v, cs[i].table, outs[i], starts[i], cs[i].n_rows, page, H, Hkv, d, ws,
                      w_in=ws_w[i], w_out=w_outs[i])

    want = []
    for i in (0, 1):
        call(i)
        want.append((outs[i].clone(), w_outs[i].clone()))
    graphs = []
    for i in (0, 1):
        graphs.append(gpu.cuda.CUDAGraph())
        gpu.cuda.synchronize()
        with gpu.cuda.graph(graphs[i]):
            call(i)
    for i in (0, 1, 1, 0, 1, 0):
        outs[i].zero_()
        w_outs[i].zero_()
        graphs[i].replay()
        gpu.cuda.synchronize()
        assert gpu.equal(outs[i], want[i][0]) and gpu.equal(w_outs[i], want[i][1])


def test_captured_and_replayed(gpu, zt):
    """A step (append, attend with weights, evict to other pages) as one graph: replays with new contents in the same
    buffers give what eager calls give."""
    H, Hkv, d, page, B, n, budget = 8, 2, 64, 16, 3, 400, 128
    rng = np.random.default_rng(15)
    c = Cache(gpu, rng, [n] * B + [budget] * B, page, Hkv, d)
    table, table_out = c.table[:B].contiguous(), c.table[B:].contiguous()
    q_start = list(range(B + 1))
    need = zt.attn_paged_workspace_bytes(q_start, [n] * B, H, Hkv, d, True)
    ws = gpu.empty(need + 16, device="cuda", dtype=gpu.uint8)
    q, kn, vn = (gpu.empty(B, h, d, device="cuda") for h in (H, Hkv, Hkv))
    q_out, out = gpu.empty_like(q), gpu.empty_like(q)
    w, w_out, w_kept = (gpu.zeros(B, Hkv, n, device="cuda") for _ in range(3))
    kept = gpu.empty(B, Hkv, budget, device="cuda", dtype=gpu.int32)

    def step():
        zt.paged_append(q, kn, vn, q_out, c.k, c.v, table, q_start, [n] * B, [n + 9] * B, page, H, Hkv, d, w=w)
        zt.attn_paged(q_out, c.k, c.v, table, out, q_start, [n] * B, page, H, Hkv, d, ws, w_in=w, w_out=w_out)
        zt.paged_evict(c.k, c.v, table, table_out, w_out, w_kept, kept, [n] * B, page, Hkv, d, 2, 16, budget)

    def fill(seed):
        gen = gpu.Generator(device="cuda").manual_seed(seed)
        for t in (q, kn, vn, w):
            t.normal_(generator=gen)

    def state():
        return [t.clone() for t in (q_out, out, w_out, w_kept, kept, c.k, c.v)]

    fill(0)
    step()  # loads the code objects
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        step()
    def clean():  # rows that no call writes keep what they hold: the same before both
        for t in (q_out, out, w_out, w_kept):
            t.fill_(-1.0)
        kept.fill_(-9)
        ws.fill_(255)

    for seed in (1, 2, 3):
        clean()
        fill(seed)
        step()
        want = state()
        clean()
        fill(seed)
        graph.replay()
        gpu.cuda.synchronize()
        for x, y in zip(want, state()):
            assert gpu.equal(x, y)


@pytest.mark.parametrize("H,Hkv,d,page", [(8, 2, 64, 16), (4, 2, 32, 4), (6, 1, 50, 8)])
def test_a_serving_run(gpu, zt, H, Hkv, d, page):
    """Prompts of two sequences, then tokens, with an eviction whenever the cache passes its limit: every output against
    64-bit attention over the rows that each head has kept."""
    rng = np.random.default_rng([H, d])
    B, budget, limit, first, last, theta = 2, 48, 64, 2, 8, 10000.0
    pages = limit // page
    pool = Cache(gpu, rng, [limit] * B, page, Hkv, d)
    w = gpu.zeros(B, Hkv, limit, device="cuda")
    kept = gpu.empty(B, Hkv, budget, device="cuda", dtype=gpu.int32)
    assert pool.table.shape[1] == pages
    n, pos = [0, 0], [0, 0]
    # What each head of each sequence holds, in 64 bits.
    k_ref = [[np.zeros((0, d)) for _ in range(Hkv)] for _ in range(B)]
    v_ref = [[np.zeros((0, d)) for _ in range(Hkv)] for _ in range(B)]
    for step in range(30):
        q_len = [37, 22] if step == 0 else [1, [0, 1, 3][step % 3]]
        n = [x + l for x, l in zip(n, q_len)]
        q_start = np.cumsum([0] + q_len).tolist()
        N = q_start[-1]
        q, kn, vn = (rng.standard_normal((N, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
        dq, dk, dv = (gpu.from_numpy(x).cuda() for x in (q, kn, vn))
        out = gpu.empty_like(dq)
        zt.paged_append(dq, dk, dv, dq, pool.k, pool.v, pool.table, q_start, n, pos, page, H, Hkv, d, theta, w)
        need = zt.attn_paged_workspace_bytes(q_start, n, H, Hkv, d, True)
        ws = gpu.empty(need + 16, device="cuda", dtype=gpu.uint8)
        zt.attn_paged(dq, pool.k, pool.v, pool.table, out, q_start, n, page, H, Hkv, d, ws, w_in=w, w_out=w)
        got = out.cpu().numpy()
        for b in range(B):
            t0, t1 = q_start[b], q_start[b + 1]
            if t1 == t0:
                continue
            qr, kr = pagedref.rotate(q[t0:t1], pos[b], theta), pagedref.rotate(kn[t0:t1], pos[b], theta)
            k1, v1 = np.zeros((n[b], Hkv, d)), np.zeros((n[b], Hkv, d))
            for h in range(Hkv):
                k_ref[b][h] = np.concatenate((k_ref[b][h], kr[:, h]))
                v_ref[b][h] = np.concatenate((v_ref[b][h], vn[t0:t1, h]))
                k1[:, h], v1[:, h] = k_ref[b][h], v_ref[b][h]
            want, _, _, bound, _ = pagedref.attend(qr, k1, v1, np.arange(n[b])[None], [0, t1 - t0], [n[b]], 1, H, Hkv, d)
            # q and k are rounded once to f32 here: their part of a score's error is as large as one product's rounding each.
            assert np.all(np.abs(got[t0:t1] - want) <= 2 * bound)
        pos = [p + l for p, l in zip(pos, q_len)]
        if max(n) + 3 > limit:
            weights = w.cpu().numpy()
            zt.paged_evict(pool.k, pool.v, pool.table, pool.table, w, w, kept, n, page, Hkv, d, first, last, budget)
            rows = kept.cpu().numpy()
            for b in range(B):
                for h in range(Hkv):
                    want = pagedref.evict(weights[b, h], n[b], budget, first, last)
                    assert np.array_equal(rows[b, h][:len(want)], want)
                    k_ref[b][h], v_ref[b][h] = k_ref[b][h][want], v_ref[b][h][want]
            n = [min(x, budget) for x in n]
    assert pos[0] > limit  # it did evict


@pytest.mark.parametrize("scores", [0, 1])
@pytest.mark.parametrize("L", [12, 40, 150])
@pytest.mark.parametrize("H,Hkv,d", [(4, 2, 32), (8, 2, 64), (6, 2, 50), (8, 2, 128), (4, 1, 192), (4, 1, 256)])
def test_a_page_of_no_pool_beside_large_values(gpu, zt, tune, H, Hkv, d, L, scores):
    """The 32-key tile of the page's keys holds a K value past 2^40 too, and a few query rows hold one: every row that
    sees the page is NaN, those with ordinary values among them; the rest, and the other sequence, as without it."""
    page, n, bad, big = 8, 200, 23, np.float32(2.0 ** 45)
    first = bad * page  # rows 184 .. 191 have no page; the large key is row 168, of the tile 160 .. 191
    rng = np.random.default_rng([H, d, L])
    c = Cache(gpu, rng, [n, n], page, Hkv, d)
    q = rng.standard_normal((2 * L, H, d)).astype(np.float32)
    q[:, :, 5] /= big
    c.k_h[pagedref.places(c.table_h, 1, n, page)[168], :, 5] *= big
    q[1::7, :, d - 2] *= big
    c.k_h[:, :, d - 2] /= big
    c.k = gpu.from_numpy(c.k_h).cuda()
    q_start, w = [0, L, 2 * L], np.zeros((2, Hkv, n), np.float32)
    tune({"ZT_PAGED_SCORES": scores})
    good = run_attend(gpu, zt, c, q, q_start, H, w)
    assert all(np.all(np.isfinite(x)) for x in good)
    c.table[1, bad] = c.n_pages
    out, lse, w1 = run_attend(gpu, zt, c, q, q_start, H, w)
    see = L + max(0, first - (n - L))  # the first token that sees the page
    assert np.array_equal(out[:see], good[0][:see]) and np.array_equal(lse[:see], good[1][:see])
    assert np.all(np.isnan(out[see:])) and np.all(np.isnan(lse[see:]))
    assert np.array_equal(w1[0], good[2][0]) and np.all(np.isnan(w1[1]))


def test_eviction_of_a_long_sequence_among_short_ones(gpu, zt):
    """64 sequences, one of 262200 rows: a workgroup for each row of the longest, had every sequence as many, would be
    more than a launch takes.  Only the first and the last page of the long one are there."""
    B, Hkv, d, page, n, budget, drop = 64, 9, 256, 64, 262200, 262190, (100, 110)
    n_rows = [5] * B
    n_rows[37] = n
    stride = -(-n // page)
    pages = 2 * (B + 1)  # in and out, two of the long sequence
    k, v = (gpu.randn(pages * page, Hkv, d, device="cuda") for _ in range(2))
    tables = []
    for at in (0, B + 1):
        t = gpu.full((B, stride), -1, dtype=gpu.int32)
        t[:, 0] = at + gpu.arange(B, dtype=gpu.int32)
        t[37, stride - 1] = at + B
        tables.append(t.cuda())
    w = gpu.ones(B, Hkv, n, device="cuda")
    w[37, :, drop[0]:drop[1]] = 0
    kept = gpu.full((B, Hkv, budget), -7, device="cuda", dtype=gpu.int32)
    want_k, want_v = k.clone(), v.clone()
    zt.paged_evict(k, v, *tables, w, w, kept, n_rows, page, Hkv, d, 0, 0, budget)
    stay = gpu.cat((gpu.arange(drop[0]), gpu.arange(drop[1], n))).int().cuda()
    for b in range(B):
        if b == 37:
            assert gpu.equal(kept[b], stay.expand(Hkv, budget)) and gpu.all(w[b, :, :budget] == 1)
        else:
            assert gpu.equal(kept[b, :, :5], gpu.arange(5, device="cuda", dtype=gpu.int32).expand(Hkv, 5))
            assert gpu.all(kept[b, :, 5:] == -1)
    out0, tail0 = (B + 1) * page, (stride - 1) * page  # the copies' first row; the last page's first
    for x, y in ((want_k, k), (want_v, v)):
        for b in range(B):
            m = page if b == 37 else 5
            x[out0 + b * page:out0 + b * page + m] = x[b * page:b * page + m]
        gone, m = drop[1] - drop[0], budget - tail0  # rows of the last page that get one of the same page
        x[out0 + B * page:out0 + B * page + m] = x[B * page + gone:B * page + gone + m]
        assert gpu.equal(x, y)


def test_append_of_more_tokens_than_one_launch_takes(gpu, zt):
    """2^25 + 77 tokens of d = 256, two to a workgroup.  Only the first and the last page are there."""
    Hkv, d, page, N = 1, 256, 1024, (1 << 25) + 77
    table = gpu.full((1, -(-N // page)), -1, device="cuda", dtype=gpu.int32)
    table[0, 0], table[0, -1] = 1, 0
    pool_k, pool_v = (gpu.zeros(2 * page, Hkv, d, device="cuda") for _ in range(2))
    new = gpu.empty(N, Hkv, d, device="cuda")
    new[:page].normal_()
    new[-77:].normal_()
    w = gpu.ones(1, Hkv, N, device="cuda")
    zt.paged_append(None, new, new, None, pool_k, pool_v, table, [0, N], [N], [0], page, 1, Hkv, d, w=w)
    assert not gpu.any(w)
    for rows, at, pos in ((new[:page], page, 0), (new[-77:], 0, N - 77)):
        n = len(rows)
        want = gpu.empty_like(rows)
        zt.rope_qk(rows.contiguous(), rows.contiguous(), want, gpu.empty_like(rows), 1, n, 1, 1, d, pos=pos)
        assert gpu.equal(pool_v[at:at + n], rows) and gpu.equal(pool_k[at:at + n], want)
    del new, rows
    gpu.cuda.empty_cache()


@pytest.mark.parametrize("d", [32, 128])
def test_weights_of_very_many_rows(gpu, zt, tune, d):
    """131072 tokens of eight heads over one, whose weight goes to the first key (0.65) and the second: sums of 2^20
    rows, formed again part by part.  All other keys have score -60.

    Tolerance, of a sum of positive terms, in half steps of f32: a weight's own error is its score's, 2 (d + 4) |s| at |s| <=
    0.62, and 24 for the exponential (2), the difference with the base (1), the row's sum (two terms, with a rescaling for
    each of a few bases, 12), its inverse (3), the product and storing (6).  A lane adds at most 128 sums of four (3 roundings)
    in 32 bits before it goes on to a wider sum, whose result is rounded once, as are those over 4 lane groups
    (2), the parts' and w_in's: 128 + 3 + 1 + 2 + 1 + 1.  The number of rows is not in it."""
    T, H, Hkv, page = 131072, 8, 1, 64
    s = np.array([np.log(0.65 / 0.35), 0.0, -60.0], np.float32)
    q0 = np.float32(np.sqrt(d))
    k = gpu.zeros(T, d, device="cuda")
    k[:, 0] = float(s[2])
    k[0, 0], k[1, 0] = float(s[0]), float(s[1])
    q = gpu.zeros(T, H * d, device="cuda")
    q.view(T, H, d)[:, :, 0] = float(q0)
    v, out = gpu.ones(T, d, device="cuda"), gpu.empty(T, H * d, device="cuda")
    table = gpu.arange(T // page, device="cuda", dtype=gpu.int32)[None].contiguous()
    w_in, w_out = gpu.zeros(1, 1, T, device="cuda"), gpu.empty(1, 1, T, device="cuda")
    tune({"ZT_PAGED_SCORES": 0})
    ws = gpu.empty(zt.attn_paged_workspace_bytes([0, T], [T], H, Hkv, d, True), device="cuda", dtype=gpu.uint8)
    zt.attn_paged(q, k, v, table, out, [0, T], [T], page, H, Hkv, d, ws, w_in=w_in, w_out=w_out)
    got = w_out[0, 0, :2].cpu().numpy().astype(np.float64)
    e = np.exp(s.astype(np.float64) * float(q0) / np.sqrt(d))
    t = np.arange(1, T)
    total = e[0] + e[1] + (t - 1) * e[2]
    want = H * np.array([1 + (e[0] / total).sum(), (e[1] / total).sum()])
    bound = (2 * (d + 4) * 0.62 + 24 + 136) * EPS
    assert np.all(np.abs(got / want - 1) <= bound), (got / want - 1, bound)


def test_the_binding_refuses_a_workspace_of_another_layout(gpu, zt):
    """An expanded tensor has as many bytes as it says nowhere."""
    H, Hkv, d, page, n = 4, 2, 32, 8, 3000
    c = Cache(gpu, np.random.default_rng(33), [n], page, Hkv, d)
    q, w = gpu.zeros(3, H * d, device="cuda"), gpu.zeros(1, Hkv, n, device="cuda")
    need = zt.attn_paged_workspace_bytes([0, 3], [n], H, Hkv, d, True)
    whole = gpu.empty(2 * need, device="cuda", dtype=gpu.uint8)
    for ws in (whole[:1].expand(need), whole[::2]):
        with pytest.raises(ValueError, match="workspace"):
            zt.attn_paged(q, c.k, c.v, c.table, gpu.empty_like(q), [0, 3], [n], page, H, Hkv, d, ws, w_in=w, w_out=w)


def attend64(gpu, q, c, q_start, H):
    """pagedref.attend by whole-matrix products on the device in 64 bits, for batches too large for its loops: the same
    outputs and bounds, the weights' with the rounding of a sum over heads and tokens counted once."""
    Hkv, d, g = c.Hkv, c.d, H // c.Hkv
    N, B = len(q), len(c.n_rows)
    f64 = dict(device="cuda", dtype=gpu.float64)
    out, bound, lse = gpu.zeros(N, H, d, **f64), gpu.zeros(N, H, d, **f64), gpu.zeros(N, H, **f64)
    w, w_bound = (gpu.zeros(B, Hkv, max(c.n_rows), **f64) for _ in range(2))
    qd = gpu.from_numpy(q).cuda()
    for b, n in enumerate(c.n_rows):
        t0, t1 = q_start[b], q_start[b + 1]
        at = gpu.from_numpy(pagedref.places(c.table_h, b, n, c.page)).cuda()
        m = (gpu.arange(n - (t1 - t0), n, **f64) + 1)[:, None, None]  # keys that each token sees
        seen = gpu.ones(t1 - t0, n, device="cuda", dtype=gpu.bool).tril(n - (t1 - t0))[:, None]
        for j in range(Hkv):
            k, v = c.k[at, j].double(), c.v[at, j].double()
            x = qd[t0:t1, j * g:(j + 1) * g].double().reshape(-1, d)
            s = gpu.mm(x, k.t().contiguous()).view(t1 - t0, g, n) / np.sqrt(d)
            size = gpu.mm(x.abs(), k.abs().t().contiguous()).view(t1 - t0, g, n) / np.sqrt(d)
            s = gpu.where(seen, s, -np.inf)
            l = gpu.logsumexp(s, 2)
            p = gpu.exp(s - l[:, :, None])
            e = 2 * (d + 4) * EPS * gpu.where(seen, size, 0.0).amax(2, keepdim=True)
            rel = gpu.expm1(e) + (m + m / 16 + 32) * EPS
            out[t0:t1, j * g:(j + 1) * g] = gpu.mm(p.view(-1, n), v).view(t1 - t0, g, d)
            bound[t0:t1, j * g:(j + 1) * g] = rel * gpu.mm(p.view(-1, n), v.abs()).view(t1 - t0, g, d)
            lse[t0:t1, j * g:(j + 1) * g] = l
            w[b, j, :n] = p.sum((0, 1))
            w_bound[b, j, :n] = (rel * p).sum((0, 1)) + g * (t1 - t0) * EPS * w[b, j, :n]
    return [x.cpu().numpy() for x in (out, lse, w, bound, w_bound)]


def test_the_two_references_agree(gpu):
    H, Hkv, d, page, n_rows, q_len = 6, 2, 50, 8, [40, 7, 129], [3, 7, 17]
    rng = np.random.default_rng(41)
    c = Cache(gpu, rng, n_rows, page, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([0] + q_len).tolist()
    q = rng.standard_normal((q_start[-1], H, d)).astype(np.float32)
    *want, w_bound = pagedref.attend(q, c.k_h, c.v_h, c.table_h, q_start, n_rows, page, H, Hkv, d)
    *got, mine = attend64(gpu, q, c, q_start, H)
    for x, y in zip(want, got):
        assert np.allclose(x, y, rtol=1e-10, atol=1e-13)
    assert np.all(mine <= w_bound * (1 + 1e-10)) and np.all(mine >= w_bound / (H // Hkv))


@pytest.mark.parametrize("H,Hkv,d", pagedref.KIND_SHAPES)
def test_a_batch_of_every_kind(gpu, zt, tune, H, Hkv, d):
    """Launches of every kind beside one another in one workspace, over more sequences than one launch takes, with weights
    from kept scores and from scores formed again (test_paged.py shows that the kinds stay apart)."""
    n_rows, q_len = pagedref.batch_of_kinds(H, Hkv)
    rng = np.random.default_rng([H, d, 42])
    c = Cache(gpu, rng, n_rows, 16, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([1] + list(q_len)).tolist()
    q = rng.standard_normal((q_start[-1] + 2, H, d)).astype(np.float32)
    w = rng.random((len(n_rows), Hkv, max(n_rows) + 5), np.float32)
    ref = attend64(gpu, q, c, q_start, H)
    for scores in (0, 1):
        tune({"ZT_PAGED_SCORES": scores})
        grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)
    grade(run_attend(gpu, zt, c, q, q_start, H), ref, q_start, n_rows, Hkv)


@pytest.mark.parametrize("target", [256, 32768])
@pytest.mark.parametrize("H,Hkv,d,rows", pagedref.FEW_SHAPES)
def test_few_rows_in_fewer_and_in_more_chunks(gpu, zt, tune, H, Hkv, d, rows, target):
    """The streaming kernel's chunks and their merges, forced (test_paged.py shows that both targets reach the plan)."""
    n_rows, q_len = pagedref.batch_of_few(H, Hkv, rows)
    rng = np.random.default_rng([H, d, rows])
    c = Cache(gpu, rng, n_rows, 16, Hkv, d, garbage=np.nan)
    q_start = np.cumsum([2] + list(q_len)).tolist()
    q = rng.standard_normal((q_start[-1] + 3, H, d)).astype(np.float32)
    w = rng.random((len(n_rows), Hkv, max(n_rows) + 5), np.float32)
    ref = attend64(gpu, q, c, q_start, H)
    tune({"ZT_PAGED_WGS": target})
    grade(run_attend(gpu, zt, c, q, q_start, H, w), ref, q_start, n_rows, Hkv, w)
    grade(run_attend(gpu, zt, c, q, q_start, H), ref, q_start, n_rows, Hkv)


@pytest.mark.parametrize("kind", ["random", "odd"])
@pytest.mark.parametrize("pages_in_place", [True, False])
@pytest.mark.parametrize("n_rows,budget,first,last,Hkv,d,page", [
    ([40, 7, 33, 0, 32], 32, 4, 8, 2, 32, 1), ([2100, 1000], 700, 1, 64, 2, 34, 16), ([5000, 1500], 1300, 4, 64, 2, 96, 64),
    ([20000, 90], 9000, 1, 1, 1, 32, 16)])
def test_eviction_of_pages_and_weights_each_its_way(gpu, zt, n_rows, budget, first, last, Hkv, d, page, pages_in_place, kind):
    """Pages in place and weights to another buffer, and the other way round."""
    rng = np.random.default_rng([len(n_rows), budget, d, 1])
    B, stride = len(n_rows), max(n_rows) + 3
    c = Cache(gpu, rng, n_rows + [budget] * B, page, Hkv, d)
    table = c.table[:B].contiguous()
    table_out, out_h = (table, c.table_h[:B]) if pages_in_place else (c.table[B:].contiguous(), c.table_h[B:])
    w = _weights(rng, B, Hkv, stride, kind)
    w_in = gpu.from_numpy(w.copy()).cuda()
    w_out = gpu.full_like(w_in, -7.0) if pages_in_place else w_in
    kept = gpu.full((B, Hkv, budget), 12345, device="cuda", dtype=gpu.int32)
    zt.paged_evict(c.k, c.v, table, table_out, w_in, w_out, kept, n_rows, page, Hkv, d, first, last, budget)
    k, v, kept_want = c.k_h.copy(), c.v_h.copy(), np.full((B, Hkv, budget), -1)
    w_want = np.full_like(w, -7.0) if pages_in_place else w.copy()
    for b, n in enumerate(n_rows):
        src, dst = pagedref.places(c.table_h, b, n, page), pagedref.places(out_h, b, min(n, budget), page)
        for h in range(Hkv):
            rows = pagedref.evict(w[b, h], n, budget, first, last)
            kept_want[b, h, :len(rows)] = rows
            k[dst, h], v[dst, h] = c.k_h[src[rows], h], c.v_h[src[rows], h]
            w_want[b, h, :len(rows)] = w[b, h, rows]
    assert np.array_equal(kept.cpu().numpy(), kept_want)
    assert np.array_equal(c.k.cpu().numpy(), k) and np.array_equal(c.v.cpu().numpy(), v)
    assert np.array_equal(w_out.cpu().numpy().view(np.uint32), w_want.view(np.uint32))
    if pages_in_place:
        assert np.array_equal(w_in.cpu().numpy().view(np.uint32), w.view(np.uint32))
