"""The paged cache's entry points without a GPU: every refusal comes before any device call, with its reason, and a
workspace's size follows from the lengths alone."""
import ctypes

import numpy as np
import pytest

import pagedref

N = ctypes.c_void_p(16)  # a pointer that no refused call follows


def ints(*xs):
    return (ctypes.c_int * len(xs))(*xs)


def attend(L, q_start=(0, 1, 3), n_rows=(5, 9), B=2, n_pages=8, page=4, stride=4, w_stride=9, H=4, Hkv=2, d=32, q=N, k=N,
           v=N, table=N, out=N, lse=None, w_in=None, w_out=None, ws=N, nbytes=1 << 40):
    return L.zt_attn_paged(q, k, v, table, out, lse, w_in, w_out, ints(*q_start) if q_start else None,
                           ints(*n_rows) if n_rows else None, B, n_pages, page, stride, w_stride, H, Hkv, d, ws, nbytes,
                           None)


def append(L, q_start=(0, 1, 3), n_rows=(5, 9), pos=(4, 7), B=2, n_pages=8, page=4, stride=4, w_stride=9, H=4, Hkv=2, d=32,
           theta=1e4, q=N, k_new=N, v_new=N, q_out=N, k=N, v=N, table=N, w=None):
    return L.zt_paged_append(q, k_new, v_new, q_out, k, v, table, w, ints(*q_start), ints(*n_rows),
                             ints(*pos) if pos else None, B, n_pages, page, stride, w_stride, H, Hkv, d, theta, None)


def evict(L, n_rows=(5, 9), B=2, n_pages=8, page=4, stride=4, w_stride=9, Hkv=2, d=32, first=1, last=2, budget=4, k=N, v=N,
          table=N, table_out=N, w_in=N, w_out=N, kept=N):
    return L.zt_paged_evict(k, v, table, table_out, w_in, w_out, kept, ints(*n_rows), B, n_pages, page, stride, w_stride,
                            Hkv, d, first, last, budget, None)


GEOMETRY = [(dict(B=0), "not launchable"), (dict(n_pages=0), "not launchable"), (dict(stride=0), "not launchable"),
            (dict(page=0), "power of two"), (dict(page=3), "power of two"), (dict(page=2048), "power of two"),
            (dict(page=-4), "power of two"), (dict(n_pages=1 << 21, page=1024), "2^31 - 1"),
            (dict(n_rows=(5, 17)), "outside [0, 16]"),
            (dict(n_rows=(5, (1 << 30) + 1), stride=1 << 21, page=1024), "outside [0, 1073741824]"), (dict(n_rows=(-1, 9)), "outside [0, 16]"),
            (dict(d=33), "head_dim"), (dict(d=300), "head_dim"), (dict(Hkv=0), "not a group")]
TOKENS = [(dict(q_start=(-1, 1, 3)), "q_start"), (dict(q_start=(0, 2, 1)), "new tokens"),
          (dict(q_start=(0, 6, 7)), "new tokens"),
          (dict(n_rows=(5, 1 << 20), stride=1 << 20, q_start=(0, 1, 1 + (1 << 20)), H=1 << 11), "new tokens"), (dict(H=3), "not a group"), (dict(H=1 << 17), "65535")]


@pytest.mark.parametrize("bad,reason", GEOMETRY + TOKENS + [
    (dict(n_rows=None), "n_rows"), (dict(q_start=None), "q_start"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(table=None), "null"), (dict(out=None), "null"), (dict(w_in=N), "together"),
    (dict(w_out=N), "together"), (dict(w_in=N, w_out=N, w_stride=8), "accumulated weights"),
    (dict(w_in=N, w_out=N, nbytes=64), "short of"), (dict(w_in=N, w_out=N, ws=None), "short of"),
    (dict(w_in=N, w_out=N, ws=ctypes.c_void_p(24)), "16-byte"), (dict(q=ctypes.c_void_p(8)), "aligned"),
    (dict(d=34, out=ctypes.c_void_p(4)), "aligned")])
def test_attend_refuses(zt, capfd, bad, reason):
    assert attend(zt.lib(), **bad) == 1
    assert reason in capfd.readouterr().err


@pytest.mark.parametrize("bad,reason", GEOMETRY + TOKENS + [
    (dict(pos=None), "pos"), (dict(pos=(-1, 0)), "position"), (dict(pos=(0, 2 ** 31 - 2)), "position"),
    (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"), (dict(q=None), "null"), (dict(q_out=None), "null"),
    (dict(k_new=None), "null"), (dict(v_new=None), "null"), (dict(k=None), "null"), (dict(table=None), "null"),
    (dict(w=N, w_stride=8), "accumulated weights"), (dict(k=ctypes.c_void_p(8)), "aligned")])
def test_append_refuses(zt, capfd, bad, reason):
    assert append(zt.lib(), **bad) == 1
    assert reason in capfd.readouterr().err


@pytest.mark.parametrize("bad,reason", GEOMETRY + [
    (dict(budget=0), "budget"), (dict(budget=(1 << 30) + 1), "budget"), (dict(first=-1), "budget"), (dict(last=-1), "budget"), (dict(first=3, last=2), "budget"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "budget"), (dict(w_stride=8), "accumulated weights"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(table=None), "null"), (dict(table_out=None), "null"),
    (dict(w_in=None), "null"), (dict(w_out=None), "null"), (dict(kept=None), "null"),
    (dict(v=ctypes.c_void_p(20)), "aligned")])
def test_evict_refuses(zt, capfd, bad, reason):
    assert evict(zt.lib(), **bad) == 1
    assert reason in capfd.readouterr().err


def test_workspace_follows_the_lengths(zt):
    L = zt.lib()

    def need(q_start, n_rows, H=32, Hkv=8, d=128, weights=0):
        return L.zt_attn_paged_workspace(ints(*q_start), ints(*n_rows), len(n_rows), H, Hkv, d, weights)

    assert need((0, 1), (16,)) == 0  # one chunk: nothing to merge
    long = need((0, 1), (1 << 20,))
    assert long > 0 and need((0, 1), (1 << 20,), weights=1) > long
    assert need((0, 1), (16,), d=33) == need((0, 2), (1,)) == need((0, 1), (-1,)) == need((0, 1), (16,), H=3) == 0
    # Chunks are of one size whatever the sequence: a batch of short sequences needs no partials.
    assert need(tuple(range(65)), (16,) * 64) == 0


def test_the_reference_agrees_with_a_dense_softmax():
    """pagedref against whole-matrix products, on a contiguous table."""
    rng = np.random.default_rng(3)
    n, L, H, Hkv, d, page = 23, 6, 6, 2, 32, 4
    k, v = rng.standard_normal((24, Hkv, d)), rng.standard_normal((24, Hkv, d))
    q = rng.standard_normal((L, H, d))
    out, lse, w, bound, w_bound = pagedref.attend(q, k, v, np.arange(6)[None], [0, L], [n], page, H, Hkv, d)
    for h in range(H):
        s = q[:, h] @ k[:n, h // 3].T / np.sqrt(d)
        s[np.arange(n)[None] > np.arange(n - L, n)[:, None]] = -np.inf
        p = np.exp(s - np.log(np.exp(s).sum(1))[:, None])
        assert np.allclose(p @ v[:n, h // 3], out[:, h], atol=1e-13)
        assert np.allclose(np.log(np.exp(s).sum(1)), lse[:, h], atol=1e-13)
        w[0, h // 3] -= p.sum(0)
    assert np.abs(w).max() < 1e-12
    assert 0 < bound.min() and bound.max() < 1e-3 and w_bound.max() < 1e-3


def test_the_reference_keeps_ties_by_row_and_nan_last():
    w = np.array([9, 1, 2, np.nan, 2, 2, -np.inf, 9, 9], np.float32)
    assert pagedref.evict(w, 9, 5, 1, 2).tolist() == [0, 2, 4, 7, 8]
    assert pagedref.evict(w, 9, 8, 1, 2).tolist() == [0, 1, 2, 4, 5, 6, 7, 8]
    assert pagedref.evict(w, 9, 9, 1, 2).tolist() == list(range(9))


@pytest.mark.parametrize("q_start,n_rows", [([0, 1], [(1 << 32) + 16]), ([0, (1 << 32) + 1], [16]), ([0, 1], [1 << 31]),
                                            ([0, 1], [-(1 << 31) - 1])])
def test_the_binding_does_not_wrap_lengths(zt, q_start, n_rows):
    with pytest.raises(ValueError, match="32 bits"):
        zt.attn_paged_workspace_bytes(q_start, n_rows, 4, 2, 32)


def test_the_binding_does_not_wrap_heads(zt):
    for bad in (((1 << 32) + 4, 2, 32), (4, (1 << 32) + 2, 32), (4, 2, (1 << 32) + 32)):
        with pytest.raises(ValueError, match="32 bits"):
            zt.attn_paged_workspace_bytes([0, 1], [16], *bad)


@pytest.mark.parametrize("page,Hkv,d", [(0, 2, 32), (8, 0, 32), (8, 2, 0), (-8, -2, 32)])
def test_the_binding_refuses_empty_pages(zt, page, Hkv, d):
    class Pool:
        def numel(self):
            return 512

    with pytest.raises(ValueError, match="holds nothing"):
        zt._paged_shapes((0,), Hkv, d, page, Pool(), Pool(), [], None, 1)


@pytest.mark.parametrize("B", [2, 8, 16])
def test_scores_past_64_bits_are_refused(zt, capfd, B):
    """2^25 tokens of 32 heads over 2^30 rows are 2^60 scores a sequence: two are counted, eight have no number."""
    q_start, n_rows = [b << 25 for b in range(B + 1)], [1 << 30] * B
    need = zt.lib().zt_attn_paged_workspace(ints(*q_start), ints(*n_rows), B, 32, 8, 128, 1)
    rc = attend(zt.lib(), q_start, n_rows, B, n_pages=8, page=1024, stride=1 << 20, H=32, Hkv=8, d=128, w_stride=1 << 30,
                w_in=N, w_out=N, nbytes=64)
    assert rc == 1
    assert (need > 0) == (B == 2)
    assert ("short of" if B == 2 else "tokens x heads") in capfd.readouterr().err


def _apart(zt, n_rows, q_len, H, Hkv, d):
    """Whether the batch's workspace is its launch kinds' own added up (a kind that joins another's is cut otherwise)."""
    def need(pick):  # without weights and with
        ls = [l for l, p in zip(q_len, pick) if p]
        ns = [n for n, p in zip(n_rows, pick) if p]
        return np.array([zt.attn_paged_workspace_bytes(np.cumsum([0] + ls), ns, H, Hkv, d, w) for w in (False, True)])

    of = [pagedref.rows_kind(l * (H // Hkv), d) for l in q_len]
    own = [need([x == kind for x in of]) for kind in sorted(set(of))]
    assert np.all(np.array(own) > 0)  # each is cut into key chunks
    return bool(np.all(need([True] * len(of)) == sum(own))), len(own)


@pytest.mark.parametrize("H,Hkv,d", pagedref.KIND_SHAPES)
def test_a_batch_of_every_kind(zt, H, Hkv, d):
    """pagedref.batch_of_kinds has launches of every kind beside one another (its figures: test_gpu_paged.py)."""
    n_rows, q_len = pagedref.batch_of_kinds(H, Hkv)
    assert _apart(zt, n_rows, q_len, H, Hkv, d) == (True, 5 if d <= 128 else 3 if d <= 192 else 2)


def test_a_short_batch_is_not_one(zt):
    """What the sum above would look like were the kinds joined."""
    assert not _apart(zt, [700, 900], [1, 90], 8, 2, 128)[0]


@pytest.mark.parametrize("H,Hkv,d,rows", pagedref.FEW_SHAPES)
def test_the_workgroup_target_reaches_the_plan(zt, tune, H, Hkv, d, rows):
    """pagedref.batch_of_few is cut into other chunks for one target than for the other."""
    n_rows, q_len = pagedref.batch_of_few(H, Hkv, rows)
    need = []
    for target in (256, 32768):
        tune({"ZT_PAGED_WGS": target})
        need.append(zt.attn_paged_workspace_bytes(np.cumsum([0] + q_len), n_rows, H, Hkv, d))
    assert 0 < need[0] < need[1]


def test_an_eviction_past_a_launch_is_refused(zt, capfd):
    """2^24 + 1 rows to other pages, a workgroup each."""
    n = (1 << 24) + 1
    assert evict(zt.lib(), n_rows=(5, n), stride=1 << 15, page=1024, w_stride=n, Hkv=9, d=256, budget=n,
                 table_out=ctypes.c_void_p(32)) == 1
    assert "workgroups" in capfd.readouterr().err
