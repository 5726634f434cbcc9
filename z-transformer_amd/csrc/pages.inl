// Entry points that deal in the paged cache's pages (include/zt_attn.h): included by zt_attn.cpp behind paged.inl,
// inside its extern "C" block.

static int pages_of(int rows, int page_size) { return (int)(((long long)rows + page_size - 1) / page_size); }

// Pages of a segment: few segments, as every workgroup adds up those before its own.
static int page_segment(int n_pages) {
    int s = ZT_PAGES_SEGMENT;
    while (n_pages / s > 4096) s *= 2;
    return s;
}
static int page_segments(int n_pages) { return pages_of(n_pages, page_segment(n_pages)); }

// Columns of a fork's entries that may need a page, -1 where an entry's rows are not usable.
static long long fork_slots(const int *n_rows, const int *n_room, int n, int page_size) {
    long long slots = 0;
    for (int i = 0; i < n; ++i) {
        if (n_rows[i] < 0 || n_room[i] < n_rows[i] || n_room[i] > kPagedMost) return -1;
        slots += pages_of(n_room[i], page_size) - n_rows[i] / page_size;
    }
    return slots;
}

namespace {
// Offsets of a fork's workspace in ints: the segments' free pages from 0 on, then ...
struct ForkSpace {
    size_t fresh, rank, list, ints;
};
ForkSpace fork_space(int n, int n_pages, long long slots) {
    ForkSpace s{};
    s.fresh = (size_t)page_segments(n_pages);
    s.rank = s.fresh + (size_t)n;
    s.list = s.rank + (size_t)slots;
    s.ints = s.list + (size_t)slots;
    return s;
}
}  // namespace

size_t zt_paged_fork_workspace(const int *n_rows, const int *n_room, int n, int n_pages, int page_size) {
    if (n < 1 || !n_rows || !n_room || paged_geometry("paged_fork_workspace", 1, n_pages, page_size, 1)) return 0;
    const long long slots = fork_slots(n_rows, n_room, n, page_size);
    return slots < 0 || slots > INT32_MAX ? 0 : fork_space(n, n_pages, slots).ints * sizeof(int);
}

int zt_paged_fork(int *table, int *refs, int *pairs, int *missing, const int *src, const int *dst, const int *n_rows,
                  const int *n_room, int n, int B, int n_pages, int page_size, int table_stride, void *workspace,
                  size_t workspace_bytes, hipStream_t stream) {
    if (paged_geometry("paged_fork", B, n_pages, page_size, table_stride)) return 1;
    if (n < 1 || n > B || !src || !dst || !n_rows || !n_room) {
        fprintf(stderr, "zt_attn: paged_fork of %d among %d sequences needs the host src, dst, n_rows and n_room arrays.\n", n,
                B);
        return 1;
    }
    const long long most = std::min((long long)table_stride * page_size, kPagedMost);
    const std::unique_ptr<unsigned char[]> to(new (std::nothrow) unsigned char[B]());
    if (!to) {
        fprintf(stderr, "zt_attn: paged_fork: no memory for %d sequences.\n", B);
        return 1;
    }
    for (int i = 0; i < n; ++i) {
        if (src[i] < 0 || src[i] >= B || dst[i] < 0 || dst[i] >= B) {
            fprintf(stderr, "zt_attn: paged_fork from sequence %d to %d, outside [0, %d).\n", src[i], dst[i], B);
            return 1;
        }
        if (n_rows[i] < 0 || n_room[i] < n_rows[i] || n_room[i] > most) {
            fprintf(stderr, "zt_attn: paged_fork of %d rows with room for %d, beyond [0, %lld].\n", n_rows[i], n_room[i], most);
            return 1;
        }
        if (to[dst[i]]++) {
            fprintf(stderr, "zt_attn: paged_fork names sequence %d twice as one that goes on.\n", dst[i]);
            return 1;
        }
    }
    for (int i = 0; i < n; ++i) {
        if (src[i] != dst[i] && to[src[i]]) {
            fprintf(stderr, "zt_attn: paged_fork from sequence %d, which the same call changes.\n", src[i]);
            return 1;
        }
    }
    const long long slots = fork_slots(n_rows, n_room, n, page_size);
    if (slots > INT32_MAX) {
        fprintf(stderr, "zt_attn: paged_fork of %lld pages is not launchable.\n", slots);
        return 1;
    }
    const ForkSpace space = fork_space(n, n_pages, slots);
    if (!workspace || workspace_bytes < space.ints * sizeof(int)) {
        fprintf(stderr, "zt_attn: paged_fork workspace of %zu bytes is short of the %zu needed.\n", workspace_bytes,
                space.ints * sizeof(int));
        return 1;
    }
    if (!workspace_aligned(workspace, "paged_fork")) return 1;
    if (!table || !refs || !pairs || !missing) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    DeviceState *st = require_device();
    if (!st) return 1;
    int *const ws = static_cast<int *>(workspace);
    ForkArgs a{};
    a.table = table; a.refs = refs; a.missing = missing;
    a.seg_free = ws; a.entry_fresh = ws + space.fresh; a.rank = ws + space.rank; a.list = ws + space.list;
    a.n_pages = n_pages; a.table_stride = table_stride;
    while (1 << a.shift < page_size) ++a.shift;
    a.segments = page_segments(n_pages);
    a.segment = page_segment(n_pages);
    a.entries = n; a.slots = (int)slots;
    // One workgroup does a small call, up to 64 pieces of 64 columns: freeing, forking 8 entries of 21 columns and copying
    // 19.6 us, with three launches 26.6, which is their way through the host; growing 64 sequences in a pool of 16000 pages
    // 11.2 us (in one of 30000, three launches, 12.1).  With more it takes longer: 78 entries of 65 columns 16.7 us, the
    // three launches 3.8 + 3.0 + 5.1 (a pass 30.5 / 27.2).
    int widest = 1;
    for (int i = 0; i < n; ++i)
        widest = std::max(widest, src[i] == dst[i] ? pages_of(n_room[i], page_size) - n_rows[i] / page_size : table_stride);
    a.pieces = widest / 64 + (widest % 64 != 0);
    const bool one = n <= ZT_PAGES_MAXE && n_pages <= ZT_PAGES_ONE && slots <= ZT_PAGES_ONE_SLOTS && (long long)n * a.pieces <= 64;
    // Else counts for all entries, a launch for each ZT_PAGES_MAXE; the list; and what they take, in launches alike.
    for (const bool take : {false, true}) {
        long long slot = 0;
        for (int e0 = 0; e0 < n; e0 += ZT_PAGES_MAXE) {
            a.entry0 = e0;
            a.n = std::min(n - e0, ZT_PAGES_MAXE);
            a.pairs = pairs + 2 * (size_t)e0;
            for (int i = 0; i < a.n; ++i) {
                a.src[i] = src[e0 + i]; a.dst[i] = dst[e0 + i];
                a.n_rows[i] = n_rows[e0 + i]; a.n_room[i] = n_room[e0 + i];
                a.slot0[i] = (int)slot;
                slot += pages_of(a.n_room[i], page_size) - a.n_rows[i] / page_size;
            }
            if (one) return launch(st, "zt_pool_fork_one", 1u, a, stream, 1024);
            const unsigned blocks = (unsigned)a.n + (!take && e0 == 0 ? (unsigned)a.segments : 0);
            if (launch(st, take ? "zt_pool_fork" : "zt_pool_count", blocks, a, stream)) return 1;
        }
        if (!take && launch(st, "zt_pool_list", (unsigned)a.segments, a, stream)) return 1;
    }
    return 0;
}

int zt_paged_free(int *table, int *refs, const int *n_keep, int B, int n_pages, int page_size, int table_stride,
                  hipStream_t stream) {
    if (paged_geometry("paged_free", B, n_pages, page_size, table_stride)) return 1;
    if (!n_keep) {
        fprintf(stderr, "zt_attn: paged_free needs the host n_keep array.\n");
        return 1;
    }
    for (int b = 0; b < B; ++b) {
        if (n_keep[b] < 0) {
            fprintf(stderr, "zt_attn: sequence %d cannot keep %d rows.\n", b, n_keep[b]);
            return 1;
        }
    }
    if (!table || !refs) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    DeviceState *st = require_device();
    if (!st) return 1;
    FreeArgs a{};
    a.table = table; a.refs = refs; a.n_pages = n_pages; a.table_stride = table_stride;
    for (int b = 0; b < B;) {
        int n = 0, least = table_stride;
        for (; b < B && n < ZT_PAGES_MAXF; ++b) {
            const int from = pages_of(n_keep[b], page_size);
            if (from >= table_stride) continue;
            a.b[n] = b;
            a.from[n++] = from;
            least = std::min(least, from);
        }
        if (n == 0) break;
        a.blocks = (int)(((long long)table_stride - least + kThreads - 1) / kThreads);
        // As many sequences at a time as a launch has room for (one's table always has).
        const int at_once = (int)std::min<long long>(n, 0xFFFFFFFFll / kThreads / a.blocks);
        for (int i0 = 0; i0 < n; i0 += at_once) {
            const int m = std::min(at_once, n - i0);
            for (int i = 0; i0 && i < m; ++i) {
                a.b[i] = a.b[i0 + i];
                a.from[i] = a.from[i0 + i];
            }
            if (launch(st, "zt_pool_free", (unsigned)m * (unsigned)a.blocks, a, stream)) return 1;
        }
    }
    return 0;
}

size_t zt_paged_compact_workspace(int n_pages) {
    return n_pages < 1 ? 0 : ((size_t)page_segments(n_pages) + (size_t)n_pages) * sizeof(int);
}

int zt_paged_compact(const int *table, const int *refs, int *table_out, int *refs_out, int *pairs, int *moved,
                     int max_pairs, int B, int n_pages, int table_stride, void *workspace, size_t workspace_bytes,
                     hipStream_t stream) {
    if (paged_geometry("paged_compact", B, n_pages, 1, table_stride)) return 1;
    if (max_pairs < 1 || max_pairs > kPagedMost) {
        fprintf(stderr, "zt_attn: paged_compact of at most %d pages is not launchable.\n", max_pairs);
        return 1;
    }
    if (!workspace || workspace_bytes < zt_paged_compact_workspace(n_pages)) {
        fprintf(stderr, "zt_attn: paged_compact workspace of %zu bytes is short of the %zu needed.\n", workspace_bytes,
                zt_paged_compact_workspace(n_pages));
        return 1;
    }
    if (!workspace_aligned(workspace, "paged_compact")) return 1;
    if (!table || !refs || !table_out || !refs_out || !pairs || !moved) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    DeviceState *st = require_device();
    if (!st) return 1;
    CompactArgs a{};
    a.table = table; a.refs = refs; a.table_out = table_out; a.refs_out = refs_out; a.pairs = pairs; a.moved = moved;
    a.segments = page_segments(n_pages);
    a.segment = page_segment(n_pages);
    a.seg_used = static_cast<int *>(workspace); a.becomes = a.seg_used + a.segments;
    a.entries = (long long)B * table_stride;
    a.n_pages = n_pages; a.max_pairs = max_pairs;
    // One workgroup does a pool that it numbers in one go and a table of few rounds, each a trip to memory.  Measured on MI355X
    // (us, one workgroup / three launches): 96 entries and 131 pages 5.5 / 9.2, 19980 and 1000 8.8 / 10.3, 32768 and 1000 11.2 /
    // 9.1; 8192 and 16384 9.3 / 10.1, 12288 10.0 / 10.1, 16384 10.8 / 10.1, 65536 (64 tables of 1024) 19.5 / 10.1.  Pairs beyond
    // the pool's pages, which no call needs, are cleared by it or by a workgroup for each segment: 100000 with 1024
    // entries and 1000 pages 13.3 / 29.1, 4000 13.9 / 14.8, 16384 16.0 / 11.7.
    const bool one = n_pages <= ZT_PAGES_ONE && a.entries + n_pages / 2 <= 20480 && (max_pairs <= n_pages || n_pages <= 4096);
    if (one) return launch(st, "zt_pool_compact_one", 1u, a, stream, 1024);
    if (launch(st, "zt_pool_used", (unsigned)a.segments, a, stream)) return 1;
    if (launch(st, "zt_pool_pair", (unsigned)a.segments, a, stream)) return 1;
    const long long work = std::max<long long>(a.entries, n_pages);
    return launch(st, "zt_pool_move", (unsigned)std::min(1024LL, (work + kThreads - 1) / kThreads), a, stream);
}

int zt_paged_copy(float *k_pages, float *v_pages, const int *pairs, int n_pairs, int n_pages, int page_size,
                  int n_kv_heads, int dim, hipStream_t stream) {
    if (paged_geometry("paged_copy", 1, n_pages, page_size, 1)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_kv_heads, n_kv_heads)) return 1;
    if (n_pairs < 0) {
        fprintf(stderr, "zt_attn: paged_copy of %d pages is not launchable.\n", n_pairs);
        return 1;
    }
    if (n_pairs == 0) return 0;
    if (!k_pages || !v_pages || !pairs) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {k_pages, v_pages})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;
    const int n = dim % 4 == 0 ? 4 : 2;
    CopyArgs a{};
    a.k = k_pages; a.v = v_pages; a.pairs = pairs; a.n_pairs = n_pairs; a.n_pages = n_pages;
    a.page_floats = (long long)page_size * n_kv_heads * dim;
    a.pieces = (int)((a.page_floats / n + ZT_PAGES_COPY - 1) / ZT_PAGES_COPY);
    const long long items = 2LL * n_pairs * a.pieces;
    return launch(st, n == 4 ? "zt_pool_copy_4" : "zt_pool_copy_2", (unsigned)std::min(items, 1LL << 20), a, stream);
}

int zt_paged_keep(float *k_pages, float *v_pages, const int *table, const int *path, const int *count, const int *q_start,
                  const int *n_rows, int B, int n_pages, int page_size, int table_stride, int n_kv_heads, int dim,
                  hipStream_t stream) {
    if (paged_check("paged_keep", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_kv_heads, n_kv_heads)) return 1;
    if (paged_tokens_check("paged_keep", q_start, n_rows, B, n_kv_heads)) return 1;
    if (!k_pages || !v_pages || !table || (q_start[B] > q_start[0] && (!path || !count))) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {k_pages, v_pages})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;
    const int n = dim % 4 == 0 ? 4 : 2;
    KeepArgs a{};
    a.pool = page_pool(k_pages, v_pages, table, n_pages, page_size, table_stride);
    a.path = path; a.count = count; a.Hkv = n_kv_heads; a.dim = dim;
    a.blocks = (2 * n_kv_heads * (dim / n) + kThreads - 1) / kThreads;
    static_assert(ZT_PAGED_MAXB * ((2ull * 65535 * 128 + kThreads - 1) / kThreads) * kThreads <= 0xFFFFFFFFull,
                  "a launch has room for every column");
    for (int b = 0; b < B;) {
        int s = 0;
        for (; b < B && s < ZT_PAGED_MAXB; ++b) {
            const int q_len = q_start[b + 1] - q_start[b];
            if (q_len == 0) continue;
            a.b[s] = b; a.q0[s] = q_start[b]; a.q_len[s] = q_len; a.row0[s] = n_rows[b] - q_len;
            ++s;
        }
        if (s && launch(st, n == 4 ? "zt_pool_keep_4" : "zt_pool_keep_2", (unsigned)(s * a.blocks), a, stream)) return 1;
    }
    return 0;
}
