"""ctypes binding of libzt_attn.so (include/zt_attn.h, include/zt_holder.h).

Plumbing for tests and the benchmark: device memory and streams come from
torch tensors, every computation runs in the HIP library.  There is no
fallback: `lib()` raises when the library has not been built, and every
wrapper raises `ZtRefused` when the C side returns non-zero.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "_build", "libzt_attn.so")

_lib = None

# The reference C ABI's six symbols, then the extensions (include/zt_attn.h),
# then the holder's C face (include/zt_holder.h).
ABI_SYMBOLS = [
    "zt_attn_dim_ok", "zt_attn_forward_shmem", "zt_attn_bwd_dq_shmem", "zt_attn_bwd_dkdv_shmem",
    "zt_attn_forward", "zt_attn_backward",
    "zt_attn_forward_batched", "zt_attn_backward_batched", "zt_attn_bwd_dq", "zt_attn_bwd_dkdv",
    "zt_attn_decode_workspace", "zt_attn_decode", "zt_attn_decode_step_workspace", "zt_attn_decode_step",
    "zt_rmsnorm_forward", "zt_rope_forward", "zt_rope_backward", "zt_rope_qk_forward",
    "zt_rope_qk_backward", "zt_fill_normal", "zt_fill_uniform", "zt_attn_version",
    "zt_attn_lds_limit", "zt_attn_plan", "zt_attn_forward_train", "zt_attn_backward_train",
    "zt_attn_bwd_dq_train", "zt_attn_bwd_dkdv_train", "zt_attn_plan_train", "zt_calibrate",
    "zt_matmul", "zt_weight_grad", "zt_input_grad", "zt_attn_backward_train_workspace",
    "zt_attn_backward_train_ws", "zt_attn_forward_train_ws", "zt_attn_set_tuning", "zt_attn_get_tuning",
    "zt_calibrate_launch", "zt_attn_decode_noalloc", "zt_matmul_plan", "zt_product_plan",
    "zt_attn_paged_workspace", "zt_attn_paged", "zt_paged_append", "zt_paged_evict",
    "zt_tree_mask", "zt_attn_paged_tree", "zt_paged_keep", "zt_paged_fork_workspace", "zt_paged_fork", "zt_paged_free",
    "zt_paged_compact_workspace", "zt_paged_compact", "zt_paged_copy", "zt_rope_frequencies", "zt_rope_at_forward",
    "zt_rope_at_backward", "zt_paged_append_at",
]
HOLDER_SYMBOLS = [
    "zt_bytes_for", "zt_to_cint", "zt_forward_bounds", "zt_holder_init", "zt_holder_deinit",
    "zt_holder_total_bytes", "zt_holder_buffer", "zt_holder_forward", "zt_holder_forward_at",
    "zt_holder_backward", "zt_holder_upload", "zt_holder_download", "zt_holder_init_exact",
    "zt_holder_workspace_bytes", "zt_holder_forget", "zt_holder_buffer_ro",
]

# include/zt_holder.h enum zt_error
ZT_OK, ZT_DEGENERATE_SHAPE, ZT_SHAPE_TOO_LARGE, ZT_CONFIG_REFUSED, ZT_DEVICE_ALLOC_FAILED, \
    ZT_DEVICE_TRANSFER_FAILED = range(6)
ZT_QUERY_HEADED, ZT_KV_HEADED, ZT_PER_ROW = range(3)
(ZT_BUF_Q, ZT_BUF_K, ZT_BUF_V, ZT_BUF_OUT, ZT_BUF_DOUT, ZT_BUF_DQ, ZT_BUF_DK, ZT_BUF_DV, ZT_BUF_ROW_MAX,
 ZT_BUF_ROW_DEN, ZT_BUF_ROW_DEL) = range(11)


class ZtRefused(RuntimeError):
    """The C side refused a call (it printed the reason on stderr)."""


def lib():
    """The library built in-tree (z-transformer_amd/_build/libzt_attn.so), bound once."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is not built; run `python z-transformer_amd/build.py` (or __graft_entry__.build())")
        _lib = load_library(LIB_PATH)
    return _lib


def load_library(path):
    """Another build of the library (the tests' planted-defect builds) with the
    same C ABI, bound like lib() and kept separate from it."""
    L = ctypes.CDLL(path, mode=os.RTLD_LOCAL)
    P, I, Z, D, U64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_double, ctypes.c_uint64
    sig = {
        "zt_attn_dim_ok": (I, [I]),
        "zt_attn_forward_shmem": (Z, [I, I, I]),
        "zt_attn_bwd_dq_shmem": (Z, [I, I]),
        "zt_attn_bwd_dkdv_shmem": (Z, [I]),
        "zt_attn_forward": (I, [P, P, P, P, I, I, I, I, I, I, I, I, P]),
        "zt_attn_backward": (I, [P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, P]),
        "zt_attn_forward_batched": (I, [P, P, P, P, I, I, I, I, I, I, I, I, I, I, P]),
        "zt_attn_backward_batched": (I, [P, P, P, P, P, P, P, P, P, P, I, I, I, I, I, I, P]),
        "zt_attn_bwd_dq": (I, [P] * 8 + [I] * 6 + [P]),
        "zt_attn_bwd_dkdv": (I, [P] * 9 + [I] * 5 + [P]),
        "zt_attn_decode_workspace": (Z, [I, I, I, I, I]),
        "zt_attn_decode": (I, [P, P, P, P, P, I, I, I, I, I, P, Z, P]),
        "zt_attn_decode_noalloc": (I, [P, P, P, P, P, I, I, I, I, I, P]),
        "zt_attn_decode_step_workspace": (Z, [I, I, I, I, I]),
        "zt_attn_decode_step": (I, [P] * 7 + [I] * 5 + [D, P, Z, P]),
        "zt_rmsnorm_forward": (I, [P, P, P, I, I, D, P]),
        "zt_attn_forward_train": (I, [P] * 5 + [I] * 5 + [P]),
        "zt_attn_backward_train": (I, [P] * 10 + [I] * 5 + [P]),
        "zt_attn_bwd_dq_train": (I, [P] * 8 + [I] * 5 + [P]),
        "zt_attn_bwd_dkdv_train": (I, [P] * 9 + [I] * 5 + [P]),
        "zt_attn_plan_train": (I, [I] * 5 + [P, P, P, Z]),
        "zt_attn_backward_train_workspace": (Z, [I] * 5),
        "zt_attn_backward_train_ws": (I, [P] * 10 + [Z] + [I] * 6 + [P]),
        "zt_attn_forward_train_ws": (I, [P] * 6 + [Z] + [I] * 5 + [P]),
        "zt_matmul": (I, [P, P, P, I, I, I, P]),
        "zt_weight_grad": (I, [P, P, P, I, I, I, P]),
        "zt_input_grad": (I, [P, P, P, I, I, I, P]),
        "zt_matmul_plan": (I, [I, I, I, P, I]),
        "zt_product_plan": (I, [I, I, I, I, P, I]),
        "zt_attn_paged_workspace": (Z, [P, P] + [I] * 5),
        "zt_attn_paged": (I, [P] * 10 + [I] * 8 + [P, Z, P]),
        "zt_paged_append": (I, [P] * 11 + [I] * 8 + [D, P]),
        "zt_paged_evict": (I, [P] * 8 + [I] * 10 + [P]),
        "zt_tree_mask": (I, [P] * 5 + [I] * 2 + [P]),
        "zt_attn_paged_tree": (I, [P] * 9 + [I] * 8 + [P, Z, P]),
        "zt_paged_keep": (I, [P] * 7 + [I] * 6 + [P]),
        "zt_paged_fork_workspace": (Z, [P, P] + [I] * 3),
        "zt_paged_fork": (I, [P] * 8 + [I] * 5 + [P, Z, P]),
        "zt_paged_free": (I, [P] * 3 + [I] * 4 + [P]),
        "zt_paged_compact_workspace": (Z, [I]),
        "zt_paged_compact": (I, [P] * 6 + [I] * 4 + [P, Z, P]),
        "zt_paged_copy": (I, [P] * 3 + [I] * 5 + [P]),
        "zt_rope_frequencies": (I, [P, I, D, I, D, D, D, D]),
        "zt_rope_at_forward": (I, [P] * 6 + [I] * 6 + [D, P]),
        "zt_rope_at_backward": (I, [P] * 6 + [I] * 6 + [D, P]),
        "zt_paged_append_at": (I, [P] * 12 + [I] * 10 + [D, P]),
        "zt_calibrate": (I, [P, Z, P, Z, P, P, P]),
        "zt_calibrate_launch": (I, [ctypes.c_uint, ctypes.c_uint, I, P, P]),
        "zt_rope_forward": (I, [P, P, I, I, I, D, I, P]),
        "zt_rope_backward": (I, [P, P, I, I, I, D, I, P]),
        "zt_rope_qk_forward": (I, [P, P, P, P, I, I, I, I, I, I, D, P]),
        "zt_rope_qk_backward": (I, [P, P, P, P, I, I, I, I, I, I, D, P]),
        "zt_fill_normal": (I, [P, Z, U64, D, D, P]),
        "zt_fill_uniform": (I, [P, Z, U64, D, D, P]),
        "zt_attn_version": (ctypes.c_char_p, []),
        "zt_attn_lds_limit": (Z, []),
        "zt_attn_set_tuning": (I, [ctypes.c_char_p, I]),
        "zt_attn_get_tuning": (I, [ctypes.c_char_p]),
        "zt_attn_plan": (I, [I, I, I, I, I, I, ctypes.c_char_p, ctypes.c_char_p, ctypes.c_char_p, Z]),
        "zt_bytes_for": (I, [I, Z, Z, Z, Z, ctypes.POINTER(Z)]),
        "zt_to_cint": (I, [Z, ctypes.POINTER(I)]),
        "zt_forward_bounds": (I, [I, I, I, I]),
        "zt_holder_init": (I, [Z, Z, Z, Z, ctypes.POINTER(P)]),
        "zt_holder_init_exact": (I, [Z, Z, Z, Z, ctypes.POINTER(P)]),
        "zt_holder_workspace_bytes": (Z, [P]),
        "zt_holder_forget": (None, [P]),
        "zt_holder_deinit": (None, [P]),
        "zt_holder_total_bytes": (Z, [P]),
        "zt_holder_buffer": (P, [P, I]),
        "zt_holder_buffer_ro": (P, [P, I]),
        "zt_holder_forward": (I, [P, I, I]),
        "zt_holder_forward_at": (I, [P, I, I, I, I, I]),
        "zt_holder_backward": (I, [P, I]),
        "zt_holder_upload": (I, [P, I, P, Z]),
        "zt_holder_download": (I, [P, P, I, Z]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    return L


def set_tuning(name, value):
    """Force a kernel variant (include/zt_attn.h, zt_attn_set_tuning); -1 restores the shape rule."""
    _check(lib().zt_attn_set_tuning(name.encode(), int(value)), f"zt_attn_set_tuning({name}, {value})")


def get_tuning(name):
    return lib().zt_attn_get_tuning(name.encode())


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _check(rc, what):
    if rc != 0:
        raise ZtRefused(f"{what} refused (rc={rc})")


def _f32_cuda(*ts):
    import torch
    for t in ts:
        if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("tensors must be contiguous float32 on the GPU")


def forward(q, k, v, out, T, n_heads, n_kv_heads, dim, group_q=1, max_tile=64, q_offset=0, n_keys=None,
            B=1, kv_rows=None, stream=None):
    """zt_attn_forward (B == 1, kv_rows == n_keys) or zt_attn_forward_batched."""
    _f32_cuda(q, k, v, out)
    n_keys = T if n_keys is None else n_keys
    if B == 1 and (kv_rows is None or kv_rows == n_keys):
        rc = lib().zt_attn_forward(_ptr(q), _ptr(k), _ptr(v), _ptr(out), T, n_heads, n_kv_heads, dim, group_q,
                                   max_tile, q_offset, n_keys, _stream(stream))
    else:
        kv_rows = n_keys if kv_rows is None else kv_rows
        rc = lib().zt_attn_forward_batched(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, T, n_heads, n_kv_heads, dim,
                                           group_q, max_tile, q_offset, n_keys, kv_rows, _stream(stream))
    _check(rc, "zt_attn_forward")


def backward(q, k, v, dout, dq, dk, dv, row_max, row_den, row_del, T, n_heads, n_kv_heads, dim, max_tile=64, B=1,
             stream=None):
    _f32_cuda(q, k, v, dout, dq, dk, dv, row_max, row_den, row_del)
    if B == 1:
        rc = lib().zt_attn_backward(*map(_ptr, (q, k, v, dout, dq, dk, dv, row_max, row_den, row_del)), T, n_heads,
                                    n_kv_heads, dim, max_tile, _stream(stream))
    else:
        rc = lib().zt_attn_backward_batched(*map(_ptr, (q, k, v, dout, dq, dk, dv, row_max, row_den, row_del)), B,
                                            T, n_heads, n_kv_heads, dim, max_tile, _stream(stream))
    _check(rc, "zt_attn_backward")


def bwd_dq(q, k, v, dout, dq, row_max, row_den, row_del, T, n_heads, n_kv_heads, dim, max_tile=64, B=1,
           stream=None):
    _f32_cuda(q, k, v, dout, dq, row_max, row_den, row_del)
    _check(lib().zt_attn_bwd_dq(*map(_ptr, (q, k, v, dout, dq, row_max, row_den, row_del)), B, T, n_heads,
                                n_kv_heads, dim, max_tile, _stream(stream)), "zt_attn_bwd_dq")


def bwd_dkdv(q, k, v, dout, dk, dv, row_max, row_den, row_del, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, dout, dk, dv, row_max, row_den, row_del)
    _check(lib().zt_attn_bwd_dkdv(*map(_ptr, (q, k, v, dout, dk, dv, row_max, row_den, row_del)), B, T, n_heads,
                                  n_kv_heads, dim, _stream(stream)), "zt_attn_bwd_dkdv")


def forward_train(q, k, v, out, lse, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, out, lse)
    _check(lib().zt_attn_forward_train(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), B, T, n_heads, n_kv_heads,
                                       dim, _stream(stream)), "zt_attn_forward_train")


# include/zt_attn.h: stage flag of zt_attn_backward_train_ws, the workspace holds the forward's scores
ZT_WS_SCORES = 4


def forward_train_ws(q, k, v, out, lse, workspace, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, out, lse, workspace)
    nbytes = workspace.numel() * workspace.element_size()
    _check(lib().zt_attn_forward_train_ws(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(workspace), nbytes,
                                          B, T, n_heads, n_kv_heads, dim, _stream(stream)),
           "zt_attn_forward_train_ws")


def backward_train(q, k, v, out, dout, lse, dq, dk, dv, delta, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, out, dout, lse, dq, dk, dv, delta)
    _check(lib().zt_attn_backward_train(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(dq),
                                        _ptr(dk), _ptr(dv), _ptr(delta), B, T, n_heads, n_kv_heads, dim,
                                        _stream(stream)), "zt_attn_backward_train")


def bwd_dq_train(q, k, v, out, dout, lse, dq, delta, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, out, dout, lse, dq, delta)
    _check(lib().zt_attn_bwd_dq_train(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(dq),
                                      _ptr(delta), B, T, n_heads, n_kv_heads, dim, _stream(stream)),
           "zt_attn_bwd_dq_train")


def bwd_dkdv_train(q, k, v, out, dout, lse, delta, dk, dv, T, n_heads, n_kv_heads, dim, B=1, stream=None):
    _f32_cuda(q, k, v, out, dout, lse, delta, dk, dv)
    _check(lib().zt_attn_bwd_dkdv_train(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(delta),
                                        _ptr(dk), _ptr(dv), B, T, n_heads, n_kv_heads, dim, _stream(stream)),
           "zt_attn_bwd_dkdv_train")


def backward_train_workspace_bytes(B, T, n_heads, n_kv_heads, dim):
    return lib().zt_attn_backward_train_workspace(B, T, n_heads, n_kv_heads, dim)


def backward_train_ws(q, k, v, out, dout, lse, dq, dk, dv, workspace, T, n_heads, n_kv_heads, dim, B=1, stage=3,
                      stream=None):
    _f32_cuda(q, k, v, out, dout, lse, dq, dk, dv, workspace)
    nbytes = workspace.numel() * workspace.element_size()
    _check(lib().zt_attn_backward_train_ws(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(dq),
                                           _ptr(dk), _ptr(dv), _ptr(workspace), nbytes, B, T, n_heads, n_kv_heads,
                                           dim, stage, _stream(stream)), "zt_attn_backward_train_ws")


def plan_train(B, T, n_heads, n_kv_heads, dim):
    bufs = [ctypes.create_string_buffer(64) for _ in range(3)]
    _check(lib().zt_attn_plan_train(B, T, n_heads, n_kv_heads, dim, *bufs, 64), "zt_attn_plan_train")
    return tuple(b.value.decode() for b in bufs)


def decode_workspace_bytes(B, n_ctx, n_heads, n_kv_heads, dim):
    return lib().zt_attn_decode_workspace(B, n_ctx, n_heads, n_kv_heads, dim)


def decode(q, k_cache, v_cache, out, n_keys, B, n_ctx, n_heads, n_kv_heads, dim, workspace, stream=None):
    """n_keys: a sequence of B ints (host)."""
    _f32_cuda(q, k_cache, v_cache, out)
    arr = (ctypes.c_int * B)(*[int(x) for x in n_keys])
    nbytes = workspace.numel() * workspace.element_size()
    rc = lib().zt_attn_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), arr, B, n_ctx, n_heads, n_kv_heads,
                              dim, _ptr(workspace), nbytes, _stream(stream))
    _check(rc, "zt_attn_decode")


def decode_step_workspace_bytes(B, n_ctx, n_heads, n_kv_heads, dim):
    return lib().zt_attn_decode_step_workspace(B, n_ctx, n_heads, n_kv_heads, dim)


def decode_step(q, k_new, v_new, k_cache, v_cache, out, pos, B, n_ctx, n_heads, n_kv_heads, dim, workspace,
                theta=500000.0, stream=None):
    """pos: a sequence of B ints (host), the position each sequence appends at."""
    _f32_cuda(q, k_new, v_new, k_cache, v_cache, out)
    arr = (ctypes.c_int * B)(*[int(x) for x in pos])
    nbytes = workspace.numel() * workspace.element_size()
    rc = lib().zt_attn_decode_step(_ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache), _ptr(out), arr,
                                   B, n_ctx, n_heads, n_kv_heads, dim, theta, _ptr(workspace), nbytes,
                                   _stream(stream))
    _check(rc, "zt_attn_decode_step")


def _i32_cuda(*ts):
    import torch
    for t in ts:
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
            raise ValueError("page tables and row numbers must be contiguous int32 on the GPU")


def _here(*ts):
    """The launches go to the current device."""
    import torch
    for t in ts:
        if t is not None and t.device.index != torch.cuda.current_device():
            raise ValueError("tensors must be on the current device")


def _c_ints(*xs):
    """The C ABI's ints; ctypes alone would cut off what does not fit."""
    xs = [int(x) for x in xs]
    if xs and (min(xs) < -(1 << 31) or max(xs) >= 1 << 31):
        raise ValueError(f"{max(xs, key=abs)} does not fit 32 bits")
    return xs


def _host_ints(xs, n):
    if len(xs) != n:
        raise ValueError(f"{len(xs)} lengths where {n} are needed")
    return (ctypes.c_int * n)(*_c_ints(*xs))


def _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages, rows, w, B):
    """What the C side cannot see: that the tensors are as long as the lengths say.  Returns n_pages."""
    of_page = page_size * n_kv_heads * dim
    if page_size < 1 or n_kv_heads < 1 or dim < 1:
        raise ValueError(f"a page of {page_size} rows of {n_kv_heads} kv heads, {dim} wide, holds nothing")
    n_pages = k_pages.numel() // of_page
    if v_pages.numel() != k_pages.numel() or n_pages * of_page != k_pages.numel():
        raise ValueError("k_pages and v_pages are [n_pages, page_size, n_kv_heads * dim]")
    for t, per_token in rows:
        if t is not None and t.numel() < int(q_start[-1]) * per_token:
            raise ValueError(f"{t.numel()} values where {int(q_start[-1])} tokens have {per_token} each")
    if w is not None and (w.dim() != 3 or tuple(w.shape[:2]) != (B, n_kv_heads)):
        raise ValueError("accumulated weights are [B, n_kv_heads, rows]")
    return n_pages


def paged_append(q, k_new, v_new, q_out, k_pages, v_pages, table, q_start, n_rows, pos, page_size, n_heads, n_kv_heads,
                 dim, theta=500000.0, w=None, stream=None):
    """q_start (B + 1), n_rows, pos (B): host sequences; table [B, pages]; w [B, n_kv_heads, rows] or None.
    q and q_out may both be None."""
    _f32_cuda(k_new, v_new, k_pages, v_pages, *[t for t in (q, q_out, w) if t is not None])
    _i32_cuda(table)
    _here(q, k_new, v_new, q_out, k_pages, v_pages, table, w)
    B, table_stride = table.shape
    n_pages = _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages,
                            [(q, n_heads * dim), (q_out, n_heads * dim), (k_new, n_kv_heads * dim),
                             (v_new, n_kv_heads * dim)], w, B)
    _check(lib().zt_paged_append(*map(_ptr, (q, k_new, v_new, q_out, k_pages, v_pages, table, w)),
                                 _host_ints(q_start, B + 1), _host_ints(n_rows, B), _host_ints(pos, B),
                                 *_c_ints(B, n_pages, page_size, table_stride, 0 if w is None else w.shape[-1], n_heads,
                                          n_kv_heads, dim), theta, _stream(stream)), "zt_paged_append")


def attn_paged_workspace_bytes(q_start, n_rows, n_heads, n_kv_heads, dim, weights=False):
    B = len(n_rows)
    return lib().zt_attn_paged_workspace(_host_ints(q_start, B + 1), _host_ints(n_rows, B), B,
                                         *_c_ints(n_heads, n_kv_heads, dim), int(weights))


def attn_paged(q, k_pages, v_pages, table, out, q_start, n_rows, page_size, n_heads, n_kv_heads, dim, workspace,
               lse=None, w_in=None, w_out=None, stream=None):
    """workspace: a tensor of attn_paged_workspace_bytes(...) bytes, or None where that is 0."""
    _f32_cuda(q, k_pages, v_pages, out, *[t for t in (lse, w_in, w_out) if t is not None])
    _i32_cuda(table)
    _here(q, k_pages, v_pages, table, out, workspace, lse, w_in, w_out)
    if w_in is not None and w_out is not None and w_in.shape != w_out.shape:
        raise ValueError("w_in and w_out have the same shape")
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    B, table_stride = table.shape
    n_pages = _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages,
                            [(q, n_heads * dim), (out, n_heads * dim), (lse, n_heads)], w_out, B)
    nbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().zt_attn_paged(*map(_ptr, (q, k_pages, v_pages, table, out, lse, w_in, w_out)),
                               _host_ints(q_start, B + 1), _host_ints(n_rows, B),
                               *_c_ints(B, n_pages, page_size, table_stride, 0 if w_out is None else w_out.shape[-1],
                                        n_heads, n_kv_heads, dim), _ptr(workspace), nbytes, _stream(stream)),
           "zt_attn_paged")


def paged_evict(k_pages, v_pages, table, table_out, w_in, w_out, kept, n_rows, page_size, n_kv_heads, dim, n_first,
                n_last, budget, stream=None):
    """kept [B, n_kv_heads, budget] int32; table_out is table (in place) or a table of other pages."""
    _f32_cuda(k_pages, v_pages, w_in, w_out)
    _i32_cuda(table, table_out, kept)
    _here(k_pages, v_pages, table, table_out, w_in, w_out, kept)
    B, table_stride = table.shape
    if table_out.shape != table.shape or w_in.shape != w_out.shape or kept.numel() != B * n_kv_heads * budget:
        raise ValueError("table and table_out, and w_in and w_out, have one shape; kept is [B, n_kv_heads, budget]")
    n_pages = _paged_shapes((0,), n_kv_heads, dim, page_size, k_pages, v_pages, [], w_in, B)
    _check(lib().zt_paged_evict(*map(_ptr, (k_pages, v_pages, table, table_out, w_in, w_out, kept)),
                                _host_ints(n_rows, B),
                                *_c_ints(B, n_pages, page_size, table_stride, w_in.shape[-1], n_kv_heads, dim, n_first,
                                         n_last, budget), _stream(stream)), "zt_paged_evict")


def _masks(mask, tokens):
    """Words of a token's mask; mask [.., words] int64 (the bits of the C side's uint64)."""
    import torch
    if mask.dtype != torch.int64 or not mask.is_cuda or not mask.is_contiguous() or mask.dim() != 2:
        raise ValueError("masks must be contiguous int64 [tokens, words] on the GPU")
    if mask.shape[0] < tokens:
        raise ValueError(f"{mask.shape[0]} masks where there are {tokens} tokens")
    return mask.shape[1]


def _at_least(n, *ts):
    for t in ts:
        if t is not None and t.numel() < n:
            raise ValueError(f"{t.numel()} values where {n} are needed")


def tree_mask(parent, mask, q_start, pos_out=None, pos=None, stream=None):
    """parent int32, mask int64 [.., words], pos_out int32: packed tokens; pos: a host sequence of B ints."""
    B, N = len(q_start) - 1, int(q_start[-1])
    _i32_cuda(*[t for t in (parent, pos_out) if t is not None])
    _here(parent, mask, pos_out)
    words = _masks(mask, N)
    _at_least(N, parent, pos_out)
    _check(lib().zt_tree_mask(_ptr(parent), _ptr(mask), _ptr(pos_out), _host_ints(q_start, B + 1),
                              None if pos is None else _host_ints(pos, B), *_c_ints(B, words), _stream(stream)),
           "zt_tree_mask")


def attn_paged_tree(q, k_pages, v_pages, table, mask, out, q_start, n_rows, page_size, n_heads, n_kv_heads, dim, workspace,
                    lse=None, stream=None):
    """workspace: a tensor of attn_paged_workspace_bytes(...) bytes, or None where that is 0."""
    _f32_cuda(q, k_pages, v_pages, out, *[t for t in (lse,) if t is not None])
    _i32_cuda(table)
    _here(q, k_pages, v_pages, table, mask, out, workspace, lse)
    words = _masks(mask, int(q_start[-1]))
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    B, table_stride = table.shape
    n_pages = _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages,
                            [(q, n_heads * dim), (out, n_heads * dim), (lse, n_heads)], None, B)
    nbytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _check(lib().zt_attn_paged_tree(*map(_ptr, (q, k_pages, v_pages, table, mask, out, lse)), _host_ints(q_start, B + 1),
                                    _host_ints(n_rows, B),
                                    *_c_ints(B, n_pages, page_size, table_stride, words, n_heads, n_kv_heads, dim),
                                    _ptr(workspace), nbytes, _stream(stream)), "zt_attn_paged_tree")


def paged_keep(k_pages, v_pages, table, path, count, q_start, n_rows, page_size, n_kv_heads, dim, stream=None):
    """path int32 [.., packed tokens], count int32 [B]."""
    _f32_cuda(k_pages, v_pages)
    _i32_cuda(table, path, count)
    _here(k_pages, v_pages, table, path, count)
    B, table_stride = table.shape
    n_pages = _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages, [(path, 1)], None, B)
    _at_least(B, count)
    _check(lib().zt_paged_keep(*map(_ptr, (k_pages, v_pages, table, path, count)), _host_ints(q_start, B + 1),
                               _host_ints(n_rows, B), *_c_ints(B, n_pages, page_size, table_stride, n_kv_heads, dim),
                               _stream(stream)), "zt_paged_keep")


def paged_fork_workspace_bytes(n_rows, n_room, n_pages, page_size):
    n = len(n_rows)
    return lib().zt_paged_fork_workspace(_host_ints(n_rows, n), _host_ints(n_room, n), *_c_ints(n, n_pages, page_size))


def paged_fork(table, refs, pairs, missing, src, dst, n_rows, n_room, page_size, workspace, stream=None):
    """table [B, pages], refs [n_pages], pairs [n, 2], missing [1]: int32; src, dst, n_rows, n_room: host sequences of n."""
    _i32_cuda(table, refs, pairs, missing)
    _here(table, refs, pairs, missing, workspace)
    if not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    (B, table_stride), n = table.shape, len(src)
    _at_least(2 * n, pairs)
    _at_least(1, missing)
    _check(lib().zt_paged_fork(*map(_ptr, (table, refs, pairs, missing)), *[_host_ints(x, n) for x in (src, dst, n_rows, n_room)],
                               *_c_ints(n, B, refs.numel(), page_size, table_stride), _ptr(workspace),
                               workspace.numel() * workspace.element_size(), _stream(stream)), "zt_paged_fork")


def paged_free(table, refs, n_keep, page_size, stream=None):
    """n_keep: a host sequence of B ints."""
    _i32_cuda(table, refs)
    _here(table, refs)
    B, table_stride = table.shape
    _check(lib().zt_paged_free(_ptr(table), _ptr(refs), _host_ints(n_keep, B),
                               *_c_ints(B, refs.numel(), page_size, table_stride), _stream(stream)), "zt_paged_free")


def paged_compact_workspace_bytes(n_pages):
    return lib().zt_paged_compact_workspace(*_c_ints(n_pages))


def paged_compact(table, refs, table_out, refs_out, pairs, moved, workspace, stream=None):
    """pairs [most, 2], moved [2] int32; table_out and refs_out are table and refs, or buffers of their own."""
    _i32_cuda(table, refs, table_out, refs_out, pairs, moved)
    _here(table, refs, table_out, refs_out, pairs, moved, workspace)
    if table_out.shape != table.shape or refs_out.shape != refs.shape or pairs.dim() != 2 or pairs.shape[1] != 2:
        raise ValueError("table and table_out, and refs and refs_out, have one shape; pairs is [most, 2]")
    if not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    _at_least(2, moved)
    B, table_stride = table.shape
    _check(lib().zt_paged_compact(*map(_ptr, (table, refs, table_out, refs_out, pairs, moved)),
                                  *_c_ints(pairs.shape[0], B, refs.numel(), table_stride), _ptr(workspace),
                                  workspace.numel() * workspace.element_size(), _stream(stream)), "zt_paged_compact")


def paged_copy(k_pages, v_pages, pairs, page_size, n_kv_heads, dim, stream=None):
    """pairs [n, 2] int32."""
    _f32_cuda(k_pages, v_pages)
    _i32_cuda(pairs)
    _here(k_pages, v_pages, pairs)
    if pairs.dim() != 2 or pairs.shape[1] != 2:
        raise ValueError("pairs is [n, 2]")
    n_pages = _paged_shapes((0,), n_kv_heads, dim, page_size, k_pages, v_pages, [], None, 1)
    _check(lib().zt_paged_copy(*map(_ptr, (k_pages, v_pages, pairs)),
                               *_c_ints(pairs.shape[0], n_pages, page_size, n_kv_heads, dim), _stream(stream)), "zt_paged_copy")


ZT_ROPE_PLAIN, ZT_ROPE_LINEAR, ZT_ROPE_BASE, ZT_ROPE_TURNS = range(4)


def rope_frequencies(rot_dim, theta=500000.0, scaling=ZT_ROPE_PLAIN, factor=1.0, low=1.0, high=4.0, context=8192.0):
    """The angle per position of each pair, a host array of rot_dim / 2 doubles."""
    rot_dim, scaling = _c_ints(rot_dim, scaling)
    freq = (ctypes.c_double * min(max(1, rot_dim // 2), 128))()  # (the C side refuses more)
    _check(lib().zt_rope_frequencies(freq, rot_dim, theta, scaling, factor, low, high, context), "zt_rope_frequencies")
    return freq


def _host_freq(freq, rot_dim):
    if len(freq) < rot_dim // 2:
        raise ValueError(f"{len(freq)} frequencies for {rot_dim} rotated columns")
    return (ctypes.c_double * len(freq))(*[float(f) for f in freq])


def rope_at(q, k, q_out, k_out, pos, freq, n_heads, n_kv_heads, head_dim, rot_dim, interleaved=False, amplitude=1.0,
            backward=False, stream=None):
    """pos [rows] int32; freq: rope_frequencies(...), or any host sequence; q or k may be None with its heads 0."""
    _f32_cuda(*[t for t in (q, k, q_out, k_out) if t is not None])
    _i32_cuda(pos)
    _here(q, k, q_out, k_out, pos)
    rows = pos.numel()
    _at_least(rows * n_heads * head_dim, q, q_out)
    _at_least(rows * n_kv_heads * head_dim, k, k_out)
    fn = lib().zt_rope_at_backward if backward else lib().zt_rope_at_forward
    _check(fn(*map(_ptr, (q, k, q_out, k_out, pos)), _host_freq(freq, rot_dim),
              *_c_ints(rows, n_heads, n_kv_heads, head_dim, rot_dim, interleaved), amplitude, _stream(stream)), "zt_rope_at")


def paged_append_at(q, k_new, v_new, q_out, k_pages, v_pages, table, pos, freq, q_start, n_rows, page_size, n_heads,
                    n_kv_heads, dim, rot_dim, interleaved=False, amplitude=1.0, w=None, stream=None):
    """paged_append at positions of each token's own: pos int32, packed tokens."""
    _f32_cuda(k_new, v_new, k_pages, v_pages, *[t for t in (q, q_out, w) if t is not None])
    _i32_cuda(table, pos)
    _here(q, k_new, v_new, q_out, k_pages, v_pages, table, pos, w)
    B, table_stride = table.shape
    n_pages = _paged_shapes(q_start, n_kv_heads, dim, page_size, k_pages, v_pages,
                            [(q, n_heads * dim), (q_out, n_heads * dim), (k_new, n_kv_heads * dim),
                             (v_new, n_kv_heads * dim), (pos, 1)], w, B)
    _check(lib().zt_paged_append_at(*map(_ptr, (q, k_new, v_new, q_out, k_pages, v_pages, table, w, pos)),
                                    _host_freq(freq, rot_dim), _host_ints(q_start, B + 1), _host_ints(n_rows, B),
                                    *_c_ints(B, n_pages, page_size, table_stride, 0 if w is None else w.shape[-1], n_heads,
                                             n_kv_heads, dim, rot_dim, interleaved), amplitude, _stream(stream)),
           "zt_paged_append_at")


def rmsnorm(x, w, y, rows, cols, eps=1e-5, stream=None):
    _f32_cuda(x, w, y)
    _check(lib().zt_rmsnorm_forward(_ptr(x), _ptr(w), _ptr(y), rows, cols, eps, _stream(stream)), "zt_rmsnorm_forward")


def rope(x, y, rows, cols, pos, theta, head_dim, stream=None):
    _f32_cuda(x, y)
    _check(lib().zt_rope_forward(_ptr(x), _ptr(y), rows, cols, pos, theta, head_dim, _stream(stream)),
           "zt_rope_forward")


def plan(B, T, n_heads, n_kv_heads, dim, max_tile=64):
    """(forward, dq, dk/dv) kernel names the library launches at this shape."""
    bufs = [ctypes.create_string_buffer(64) for _ in range(3)]
    _check(lib().zt_attn_plan(B, T, n_heads, n_kv_heads, dim, max_tile, *bufs, 64), "zt_attn_plan")
    return tuple(b.value.decode() for b in bufs)


def rope_backward(dout, din, rows, cols, pos, theta, head_dim, stream=None):
    _f32_cuda(dout, din)
    _check(lib().zt_rope_backward(_ptr(dout), _ptr(din), rows, cols, pos, theta, head_dim, _stream(stream)),
           "zt_rope_backward")


def rope_qk(q, k, q_out, k_out, B, T, n_heads, n_kv_heads, head_dim, pos=0, theta=500000.0, backward=False,
            stream=None):
    _f32_cuda(q, k, q_out, k_out)
    fn = lib().zt_rope_qk_backward if backward else lib().zt_rope_qk_forward
    _check(fn(_ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), B, T, n_heads, n_kv_heads, head_dim, pos, theta,
              _stream(stream)), "zt_rope_qk")


class DimensionMismatch(ValueError):
    """src/tensor.zig:79: a.cols != b.rows."""


def matmul(a, b, out, M, K, N, stream=None):
    """out[M,N] = a[M,K] b[K,N] (src/tensor.zig:78-106)."""
    _f32_cuda(a, b, out)
    if a.numel() != M * K or b.numel() != K * N or out.numel() != M * N:
        raise DimensionMismatch(f"{M}x{K} @ {K}x{N} into {out.numel()} elements")
    _check(lib().zt_matmul(_ptr(a), _ptr(b), _ptr(out), M, K, N, _stream(stream)), "zt_matmul")


def gemm_kernel(M, K, N, product="nn"):
    """The kernel zt_matmul ("nn"), zt_weight_grad ("tn") or zt_input_grad ("nt") launches for an M x N result over K."""
    buf = ctypes.create_string_buffer(64)
    _check(lib().zt_product_plan(("nn", "tn", "nt").index(product), M, K, N, buf, 64), "zt_product_plan")
    return buf.value.decode()


def weight_grad(w, inp, dout, T, I, J, stream=None):
    """w[I,J] += inp[T,I]^T dout[T,J] (src/autograd.zig:958-972)."""
    _f32_cuda(w, inp, dout)
    _check(lib().zt_weight_grad(_ptr(w), _ptr(inp), _ptr(dout), T, I, J, _stream(stream)), "zt_weight_grad")


def input_grad(din, dout, w, T, J, I, stream=None):
    """din[T,I] += dout[T,J] w[I,J]^T (src/autograd.zig:999-1022)."""
    _f32_cuda(din, dout, w)
    _check(lib().zt_input_grad(_ptr(din), _ptr(dout), _ptr(w), T, J, I, _stream(stream)), "zt_input_grad")


def calibrate(src, scratch, stream=None):
    """(sustained FP32 MFMA TFLOP/s, streaming-read GB/s) measured on this device."""
    _f32_cuda(src, scratch)
    tf, gb = ctypes.c_double(0.0), ctypes.c_double(0.0)
    _check(lib().zt_calibrate(_ptr(src), src.numel() * 4, _ptr(scratch), scratch.numel() * 4, ctypes.addressof(tf),
                              ctypes.addressof(gb), _stream(stream)), "zt_calibrate")
    return tf.value, gb.value


def launch_floor_us(blocks, threads, launches=256, stream=None):
    """Average microseconds per back-to-back launch of an empty kernel of this grid."""
    us = ctypes.c_double(0.0)
    _check(lib().zt_calibrate_launch(blocks, threads, launches, ctypes.addressof(us), _stream(stream)),
           "zt_calibrate_launch")
    return us.value


def fill_normal(t, seed, mean=0.0, sigma=1.0, stream=None):
    _f32_cuda(t)
    _check(lib().zt_fill_normal(_ptr(t), t.numel(), seed, mean, sigma, _stream(stream)), "zt_fill_normal")


def fill_uniform(t, seed, lo=0.0, hi=1.0, stream=None):
    _f32_cuda(t)
    _check(lib().zt_fill_uniform(_ptr(t), t.numel(), seed, lo, hi, _stream(stream)), "zt_fill_uniform")
