"""Trees, rotary positions and shared pages without a GPU: every refusal comes before any device call, with its reason;
workspaces and frequencies follow from the host's numbers alone."""
import ctypes

import numpy as np
import pytest

import pagedref
import treeref

N = ctypes.c_void_p(16)  # a pointer that no refused call follows
ODD = ctypes.c_void_p(20)


def ints(xs):
    return None if xs is None else (ctypes.c_int * len(xs))(*xs)


def doubles(xs):
    return None if xs is None else (ctypes.c_double * len(xs))(*xs)


def mask(L, parent=N, out=N, pos_out=N, q_start=(0, 1, 3), pos=(4, 7), B=2, words=1):
    return L.zt_tree_mask(parent, out, pos_out, ints(q_start), ints(pos), B, words, None)


def attend(L, q_start=(0, 1, 3), n_rows=(5, 9), B=2, n_pages=8, page=4, stride=4, words=1, H=4, Hkv=2, d=32, q=N, k=N, v=N,
           table=N, masks=N, out=N, ws=N, nbytes=1 << 40):
    return L.zt_attn_paged_tree(q, k, v, table, masks, out, None, ints(q_start), ints(n_rows), B, n_pages, page, stride, words,
                                H, Hkv, d, ws, nbytes, None)


def keep(L, q_start=(0, 1, 3), n_rows=(5, 9), B=2, n_pages=8, page=4, stride=4, Hkv=2, d=32, k=N, v=N, table=N, path=N,
         count=N):
    return L.zt_paged_keep(k, v, table, path, count, ints(q_start), ints(n_rows), B, n_pages, page, stride, Hkv, d, None)


def append(L, q_start=(0, 1, 3), n_rows=(5, 9), pos=N, B=2, n_pages=8, page=4, stride=4, w_stride=9, H=4, Hkv=2, d=32, rot=32,
           inter=0, amplitude=1.0, freq=(1.0,) * 16, q=N, k_new=N, v_new=N, q_out=N, k=N, v=N, table=N, w=None):
    return L.zt_paged_append_at(q, k_new, v_new, q_out, k, v, table, w, pos, doubles(freq), ints(q_start), ints(n_rows), B,
                                n_pages, page, stride, w_stride, H, Hkv, d, rot, inter, amplitude, None)


def fork(L, src=(0, 0), dst=(1, 2), n_rows=(5, 9), n_room=(6, 9), n=2, B=4, n_pages=8, page=4, stride=4, table=N, refs=N,
         pairs=N, missing=N, ws=N, nbytes=1 << 30):
    return L.zt_paged_fork(table, refs, pairs, missing, ints(src), ints(dst), ints(n_rows), ints(n_room), n, B, n_pages, page,
                           stride, ws, nbytes, None)


def free(L, n_keep=(0, 5), B=2, n_pages=8, page=4, stride=4, table=N, refs=N):
    return L.zt_paged_free(table, refs, ints(n_keep), B, n_pages, page, stride, None)


def compact(L, B=2, n_pages=8, stride=4, most=4, table=N, refs=N, table_out=N, refs_out=N, pairs=N, moved=N, ws=N,
            nbytes=1 << 30):
    return L.zt_paged_compact(table, refs, table_out, refs_out, pairs, moved, most, B, n_pages, stride, ws, nbytes, None)


def copy(L, n_pairs=2, n_pages=8, page=4, Hkv=2, d=32, k=N, v=N, pairs=N):
    return L.zt_paged_copy(k, v, pairs, n_pairs, n_pages, page, Hkv, d, None)


def turn(L, rows=3, H=2, Hkv=1, d=32, rot=32, inter=0, amplitude=1.0, freq=(1.0,) * 16, q=N, k=N, q_out=N, k_out=N, pos=N,
         back=False):
    fn = L.zt_rope_at_backward if back else L.zt_rope_at_forward
    return fn(q, k, q_out, k_out, pos, doubles(freq), rows, H, Hkv, d, rot, inter, amplitude, None)


POOL = [(dict(B=0), "not launchable"), (dict(n_pages=0), "not launchable"), (dict(stride=0), "not launchable")]
PAGE = [(dict(page=0), "power of two"), (dict(page=3), "power of two"), (dict(page=2048), "power of two"),
        (dict(n_pages=1 << 21, page=1024), "2^31 - 1")]
ROWS = [(dict(n_rows=(5, 17)), "outside [0, 16]"), (dict(n_rows=(-1, 9)), "outside [0, 16]"), (dict(n_rows=None), "n_rows"),
        (dict(q_start=(-1, 1, 3)), "q_start"), (dict(q_start=(0, 2, 1)), "new tokens"), (dict(q_start=None), "q_start"),
        (dict(q_start=(0, 6, 7)), "new tokens"), (dict(d=33), "head_dim"), (dict(d=300), "head_dim"),
        (dict(Hkv=0), "not a group")]
TURNS = [(dict(rot=0), "rotated columns"), (dict(rot=31), "rotated columns"), (dict(rot=34), "rotated columns"),
         (dict(rot=-2), "rotated columns"), (dict(inter=2), "interleaved"), (dict(inter=-1), "interleaved"),
         (dict(freq=None), "frequencies"), (dict(amplitude=float("inf")), "amplitude"),
         (dict(amplitude=float("nan")), "amplitude"), (dict(freq=(1.0,) * 15 + (float("nan"),)), "frequency 15"),
         (dict(freq=(float("inf"),) + (1.0,) * 15), "frequency 0")]
CASES = [(mask, [(dict(B=0), "q_start"), (dict(q_start=None), "q_start"), (dict(q_start=(-1, 0, 1)), "q_start"),
                 (dict(q_start=(0, 3, 2)), "new tokens"), (dict(words=0), "64-bit words"), (dict(words=-1), "64-bit words"),
                 (dict(q_start=(0, 1, 66)), "64-bit words"), (dict(words=1 << 25), "64-bit words"),
                 (dict(pos=None), "together"), (dict(pos_out=None), "together"), (dict(pos=(-1, 0)), "position"),
                 (dict(pos=(0, 2 ** 31 - 2)), "position"), (dict(parent=None), "null"), (dict(out=None), "null"),
                 (dict(out=ODD), "8-byte")]),
         (attend, POOL + PAGE + ROWS + [
             (dict(words=0), "64-bit words"), (dict(n_rows=(5, 80), q_start=(0, 1, 66), stride=32), "64-bit words"),
             (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(table=None), "null"),
             (dict(out=None), "null"), (dict(masks=None), "null"), (dict(masks=ODD), "8-byte"), (dict(q=ODD), "aligned"),
             (dict(H=3), "not a group"), (dict(n_rows=(5, 100000), stride=32768, n_pages=1 << 15, nbytes=16), "short of"),
             (dict(n_rows=(5, 100000), stride=32768, n_pages=1 << 15, ws=None), "short of"),
             (dict(n_rows=(5, 100000), stride=32768, n_pages=1 << 15, ws=ctypes.c_void_p(24)), "16-byte")]),
         (keep, POOL + PAGE + ROWS + [(dict(k=None), "null"), (dict(v=None), "null"), (dict(table=None), "null"),
                                      (dict(path=None), "null"), (dict(count=None), "null"), (dict(v=ODD), "aligned")]),
         (append, POOL + PAGE + ROWS + TURNS + [
             (dict(pos=None), "null"), (dict(q=None), "null"), (dict(q_out=None), "null"), (dict(k_new=None), "null"),
             (dict(v_new=None), "null"), (dict(k=None), "null"), (dict(table=None), "null"), (dict(k=ODD), "aligned"),
             (dict(w=N, w_stride=8), "accumulated weights")]),
         (fork, POOL + PAGE + [
             (dict(n=0), "src, dst"), (dict(n=5), "src, dst"), (dict(src=None), "src, dst"), (dict(dst=None), "src, dst"),
             (dict(n_rows=None), "src, dst"), (dict(n_room=None), "src, dst"), (dict(src=(0, 4)), "outside [0, 4)"),
             (dict(dst=(-1, 1)), "outside [0, 4)"), (dict(n_rows=(-1, 9)), "room"), (dict(n_rows=(7, 9)), "room"),
             (dict(n_room=(6, 17)), "room"), (dict(dst=(1, 1)), "twice"), (dict(src=(0, 1)), "same call changes"),
             (dict(src=(0, 0), dst=(0, 2)), "same call changes"), (dict(ws=None), "short of"), (dict(nbytes=8), "short of"),
             (dict(ws=ctypes.c_void_p(24)), "16-byte"), (dict(table=None), "null"), (dict(refs=None), "null"),
             (dict(pairs=None), "null"), (dict(missing=None), "null")]),
         (free, POOL + PAGE + [(dict(n_keep=None), "n_keep"), (dict(n_keep=(0, -1)), "cannot keep"), (dict(table=None), "null"),
                               (dict(refs=None), "null")]),
         (compact, POOL + [(dict(most=0), "at most 0"), (dict(most=(1 << 30) + 1), "at most"), (dict(ws=None), "short of"),
                           (dict(nbytes=32), "short of"), (dict(ws=ctypes.c_void_p(24)), "16-byte")] +
          [({x: None}, "null") for x in ("table", "refs", "table_out", "refs_out", "pairs", "moved")]),
         (copy, PAGE + [(dict(n_pages=0), "not launchable"), (dict(n_pairs=-1), "not launchable"), (dict(d=33), "head_dim"),
                        (dict(Hkv=0), "not a group"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(pairs=None), "null"),
                        (dict(k=ODD), "aligned")]),
         (turn, TURNS + [(dict(back=True, **x), r) for x, r in TURNS] + [
             (dict(d=0), "head_dim"), (dict(d=33), "head_dim"), (dict(d=258), "head_dim"), (dict(rows=-1), "rows"),
             (dict(H=-1), "rows"), (dict(Hkv=-1), "rows"), (dict(H=65536), "rows"), (dict(q=None), "null"),
             (dict(k_out=None), "null"), (dict(pos=None), "null"), (dict(q_out=ODD), "aligned")])]


@pytest.mark.parametrize("call,bad,reason", [(c, b, r) for c, bads in CASES for b, r in bads])
def test_refuses(zt, capfd, call, bad, reason):
    assert call(zt.lib(), **bad) == 1
    assert reason in capfd.readouterr().err


def test_nothing_to_do_is_no_error(zt):
    L = zt.lib()
    assert turn(L, rows=0) == 0 and turn(L, H=0, Hkv=0) == 0 and copy(L, n_pairs=0) == 0


def test_workspaces_follow_the_numbers(zt):
    L = zt.lib()

    def need(n_rows, n_room, n_pages=100, page=16):
        return L.zt_paged_fork_workspace(ints(n_rows), ints(n_room), len(n_rows), n_pages, page)

    # A count per segment of 1024 pages, one per entry, two numbers per page that may be wanted.
    assert need((5,), (5,)) == 4 * (1 + 1 + 2) and need((16,), (16,)) == 4 * 2 and need((5, 16), (40, 16)) == 4 * (1 + 2 + 6)
    assert need((5,), (5,), n_pages=1025) == 4 * (2 + 1 + 2)
    assert need((5,), (4,)) == need((-1,), (4,)) == need((5,), (5,), page=3) == need((5,), (5,), n_pages=0) == 0
    assert need((0,), ((1 << 30) + 1,)) == 0
    # Past 2^22 pages segments grow, so that there are 4096 or so.
    assert need((16,), (16,), n_pages=(1 << 22) + 1024) == 4 * (2049 + 1) and need((16,), (16,), n_pages=2 ** 31 - 1, page=1) == 4 * (4096 + 1)
    assert L.zt_paged_compact_workspace(0) == 0 and L.zt_paged_compact_workspace(4097) == 4 * (5 + 4097)


@pytest.mark.parametrize("rot", [2, 4, 48, 128, 256])
@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "turns"])
def test_frequencies(zt, rot, scaling):
    number = ["plain", "linear", "base", "turns"].index(scaling)
    if scaling == "base" and rot == 2:
        with pytest.raises(zt.ZtRefused):
            zt.rope_frequencies(rot, 1e4, number, 8.0)
        return
    got = np.array(zt.rope_frequencies(rot, 500000.0, number, 8.0, 1.0, 4.0, 8192.0))
    want = treeref.frequencies(rot, 500000.0, scaling, 8.0, 1.0, 4.0, 8192.0)
    assert np.allclose(got, want, rtol=8 * 2.0 ** -53 * 20, atol=0)  # (pow: a step; its argument's, times ln theta < 20)
    plain = treeref.frequencies(rot, 500000.0)
    if scaling == "turns" and rot >= 48:
        assert got[0] == plain[0] and np.isclose(got[-1], plain[-1] / 8, rtol=1e-14)
    if scaling == "base":
        assert got[0] == 1.0 and np.isclose(got[-1], plain[-1] / 8, rtol=1e-13)


@pytest.mark.parametrize("args", [(0,), (3,), (258,), (32, 0.0), (32, float("nan")), (32, float("inf")), (32, 1e4, 4), (32, 1e4, -1),
                                  (32, 1e4, 1, 0.0), (32, 1e4, 1, float("nan")), (32, 1e4, 2, -1.0), (32, 1e4, 3, 8.0, 4.0, 4.0),
                                  (32, 1e4, 3, 8.0, 1.0, 4.0, 0.0), (32, 1e4, 3, 8.0, float("nan"), 4.0)])
def test_frequencies_refuse(zt, args):
    with pytest.raises(zt.ZtRefused):
        zt.rope_frequencies(*args)


@pytest.mark.parametrize("args", [(4, 1.0, 2, 1e-200), (4, 5e5, 2, 1e300), (32, 1e4, 1, 1e-310), (32, 1e4, 1, 5e-324),
                                  (128, 1e-320, 3, 5e-324, 1e300, 2e300, 1.0)])
def test_frequencies_beyond_64_bits_are_refused(zt, capfd, args):
    """Usable numbers by themselves, whose base or quotient is none; nothing is written."""
    freq = (ctypes.c_double * 128)(*[-7.0] * 128)
    rot, theta, scaling, factor, low, high, context = (list(args) + [1.0, 4.0, 8192.0][len(args) - 4:])[:7]
    assert zt.lib().zt_rope_frequencies(freq, rot, theta, scaling, factor, low, high, context) == 1
    assert "beyond 64 bits" in capfd.readouterr().err and set(freq) == {-7.0}
    # As far as 64 bits go they are had.
    assert zt.lib().zt_rope_frequencies(freq, 4, 5e5, 2, 1e100, 0.0, 0.0, 0.0) == 0 and 0 < freq[1] < 1e-100
    assert zt.lib().zt_rope_frequencies(freq, 4, 1e4, 1, 1e-300, 0.0, 0.0, 0.0) == 0 and np.isfinite(freq[1]) and freq[0] == 1 / 1e-300


def test_the_binding_does_not_wrap(zt):
    for call in (lambda: zt.paged_fork_workspace_bytes([1 << 32], [5], 8, 4), lambda: zt.paged_fork_workspace_bytes([5], [5], 1 << 32, 4),
                 lambda: zt.paged_compact_workspace_bytes((1 << 32) + 8), lambda: zt.rope_frequencies((1 << 32) + 32)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    with pytest.raises(ValueError, match="frequencies"):
        zt._host_freq([1.0] * 15, 32)


def test_the_reference_agrees_with_a_chunks(zt):
    """treeref against pagedref where the tree is a line."""
    rng = np.random.default_rng(3)
    n, L, H, Hkv, d, page = 23, 6, 6, 2, 32, 4
    k, v = rng.standard_normal((24, Hkv, d)), rng.standard_normal((24, Hkv, d))
    q = rng.standard_normal((L, H, d))
    table = np.arange(6)[None]
    mask, depth = treeref.masks([np.arange(-1, L - 1)], 1)
    assert depth.tolist() == list(range(L))
    want = pagedref.attend(q, k, v, table, [0, L], [n], page, H, Hkv, d)
    out, lse, bound = treeref.attend(q, k, v, table, [0, L], [n], page, H, Hkv, d, [treeref.seen(mask, n, L)])
    assert np.allclose(out, want[0], atol=1e-14) and np.allclose(lse, want[1], atol=1e-14) and bound.max() < 1e-3


def test_the_reference_of_pages_keeps_its_counts():
    rng = np.random.default_rng(4)
    p = treeref.Pages(np.full((6, 8), -1, np.int32), np.zeros(20, np.int32), 4)
    assert p.fork([0], [0], [0], [10])[1] == 0 and p.table[0].tolist() == [0, 1, 2] + [-1] * 5
    pairs, missing = p.fork([0, 0], [1, 2], [9, 8], [9, 13])
    assert missing == 0 and pairs.tolist() == [[2, 3], [-1, -1]]
    assert p.table[1, :3].tolist() == [0, 1, 3] and p.table[2, :4].tolist() == [0, 1, 4, 5]
    assert p.refs[:6].tolist() == [3, 3, 1, 1, 1, 1] and np.array_equal(p.refs, p.counted())
    # Cut back into a shared page, then grown: the page is replaced.
    p.free([6, 32, 32, 32, 32, 32])
    pairs, missing = p.fork([0], [0], [6], [7])
    assert missing == 0 and pairs.tolist() == [[1, 2]] and np.array_equal(p.refs, p.counted())
    assert p.fork([1], [3], [0], [32])[1] == 0
    assert p.fork([1], [4], [0], [32])[1] == 2
    p.free([32, 0, 32, 0, 32, 32])
    pairs, moved = p.compact(20)
    assert moved[1] == 0 and np.all(p.refs[:np.count_nonzero(p.refs)] > 0) and np.array_equal(p.refs, p.counted())
