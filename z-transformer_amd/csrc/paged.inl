// Entry points of the paged KV cache (include/zt_attn.h): included by zt_attn.cpp
// inside its extern "C" block, whose launcher, checks and device state they use.
//
// The plan of a call -- which kernel takes which sequence, in how many key chunks --
// follows from the host's lengths alone, so that a workspace's size does not depend
// on the device.

// The cache's geometry; 0 when usable.
static int paged_check(const char *who, const int *n_rows, int B, int n_pages, int page_size, int table_stride) {
    if (B < 1 || n_pages < 1 || table_stride < 1) {
        fprintf(stderr, "zt_attn: %s over %d sequences of at most %d pages in a pool of %d is not launchable.\n", who, B,
                table_stride, n_pages);
        return 1;
    }
    if (page_size < 1 || page_size > 1024 || (page_size & (page_size - 1)) != 0) {
        fprintf(stderr, "zt_attn: a page of %d rows is refused. It must hold a power of two of them in [1, 1024].\n",
                page_size);
        return 1;
    }
    if ((long long)n_pages * page_size > INT32_MAX) {
        fprintf(stderr, "zt_attn: %d pages of %d rows are more than 2^31 - 1 rows.\n", n_pages, page_size);
        return 1;
    }
    if (!n_rows) {
        fprintf(stderr, "zt_attn: %s needs the host n_rows array.\n", who);
        return 1;
    }
    for (int b = 0; b < B; ++b) {
        if (n_rows[b] < 0 || n_rows[b] > (long long)table_stride * page_size) {
            fprintf(stderr, "zt_attn: sequence %d has n_rows %d, outside [0, %lld].\n", b, n_rows[b],
                    (long long)table_stride * page_size);
            return 1;
        }
    }
    return 0;
}

// The batch's new tokens: packed in order, the last rows of their sequences.
static int paged_tokens_check(const char *who, const int *q_start, const int *n_rows, int B, int n_heads) {
    if (!q_start || q_start[0] < 0) {
        fprintf(stderr, "zt_attn: %s needs the host q_start array, from 0 up.\n", who);
        return 1;
    }
    for (int b = 0; b < B; ++b) {
        const long long q_len = (long long)q_start[b + 1] - q_start[b];
        if (q_len < 0 || q_len > n_rows[b] || q_len * n_heads > INT32_MAX) {
            fprintf(stderr, "zt_attn: sequence %d has %lld new tokens among its %d rows.\n", b, q_len, n_rows[b]);
            return 1;
        }
    }
    return 0;
}

static int paged_weights_check(const char *who, const int *n_rows, int B, int w_stride) {
    for (int b = 0; b < B; ++b) {
        if (n_rows[b] > w_stride) {
            fprintf(stderr, "zt_attn: %s: sequence %d's %d rows exceed the %d accumulated weights of a head.\n", who, b,
                    n_rows[b], w_stride);
            return 1;
        }
    }
    return 0;
}

static PagePool page_pool(float *k, float *v, const int *table, int n_pages, int page_size, int table_stride) {
    PagePool p{};
    p.k = k; p.v = v; p.table = table;
    p.n_pages = n_pages; p.table_stride = table_stride;
    while (1 << p.shift < page_size) ++p.shift;
    return p;
}

// Padded width of the paged kernels.
static int paged_dp(int dim) {
    const int dp = pad32(dim);
    return dp == 160 ? 192 : dp == 224 ? 256 : dp;
}

namespace {

// Which kernel takes a sequence, by its rows per kv head (new tokens x heads of the group): the streaming
// kernel with one or two 16-row blocks, or the split-operand one.
enum class PagedKind { None, Few1, Few2, Many };
constexpr PagedKind kPagedKinds[] = {PagedKind::Few1, PagedKind::Few2, PagedKind::Many};

// What a call does for each sequence.
struct PagedPlan {
    const int *q_start, *n_rows;
    int B, H, Hkv, G, dim, dp, part_ld;
    int chunk_few, chunk_many;  // keys of a workgroup
    int part_rows;              // rows of a part of the weights' sums (Many)

    int q_len(int b) const { return q_start[b + 1] - q_start[b]; }
    int rows(int b) const { return q_len(b) * G; }
    PagedKind kind(int b) const {
        const int r = rows(b);
        return r == 0 ? PagedKind::None : r <= 16 ? PagedKind::Few1 : r <= 32 ? PagedKind::Few2 : PagedKind::Many;
    }
    bool many(int b) const { return kind(b) == PagedKind::Many; }
    int many_rows() const { return dp <= 128 ? 256 : 128; }     // of a workgroup
    int weight_keys() const { return dp <= 128 ? 256 : 128; }   // of a workgroup of the weights' sums
    int tiles(int b) const { return many(b) ? (rows(b) + many_rows() - 1) / many_rows() : 1; }
    int chunk(int b) const { return many(b) ? chunk_many : chunk_few; }
    int chunks(int b) const { return q_len(b) ? (n_rows[b] + chunk(b) - 1) / chunk(b) : 0; }
    long long items(int b) const { return (long long)tiles(b) * chunks(b) * Hkv; }
    long long slots(int b) const { return chunks(b) > 1 ? (long long)q_len(b) * H * chunks(b) : 0; }
    int kpad(int b) const { return (n_rows[b] + 15) / 16 * 16; }
    int parts(int b) const { return (rows(b) + part_rows - 1) / part_rows; }
    // Floats that the weights need: every row's scores, or the parts' sums.
    long long scores(int b) const { return (long long)kpad(b) * (many(b) ? (long long)Hkv * parts(b) : (long long)q_len(b) * H); }
};

PagedPlan paged_plan(const int *q_start, const int *n_rows, int B, int H, int Hkv, int dim) {
    PagedPlan p{q_start, n_rows, B, H, Hkv, H / Hkv, dim, paged_dp(dim), (dim + 3) / 4 * 4, 0, 0, 0};
    long long few = 0, many = 0, most = 0, sums = 0;  // steps of 16 and of 32 keys; row tiles x key tiles
    for (int b = 0; b < B; ++b) {
        if (p.many(b)) {
            many += (long long)p.tiles(b) * Hkv * ((n_rows[b] + 31) / 32);
            most = std::max(most, (long long)(n_rows[b] + 31) / 32);
            sums += (long long)p.rows(b) * Hkv * ((n_rows[b] + p.weight_keys() - 1) / p.weight_keys());
        } else if (p.q_len(b)) {
            few += (long long)Hkv * ((n_rows[b] + 15) / 16);
        }
    }
    const long long f = std::max(8LL, (few + 1023) / 1024);
    p.chunk_few = (int)std::min(16 * ((f + 3) / 4 * 4), 1LL << 30);  // whole rounds of four waves
    const long long m = std::max(8LL, (many + 255) / 256);
    p.chunk_many = (int)std::min(32 * m, 1LL << 30);
    p.part_rows = (int)std::min(std::max(256LL, (sums / 512 + 31) / 32 * 32), 1LL << 30);
    return p;
}

// Offsets of a workspace's parts in bytes.
struct PagedSpace {
    size_t ml, stat, scores, bytes;
};
PagedSpace paged_space(const PagedPlan &p, bool weights) {
    long long slots = 0, scores = 0;
    for (int b = 0; b < p.B; ++b) {
        slots += p.slots(b);
        scores += p.scores(b);
    }
    PagedSpace s{};
    s.ml = align256((size_t)slots * p.part_ld * sizeof(float));
    s.stat = s.ml + align256((size_t)slots * 2 * sizeof(float));
    s.scores = s.stat + (weights ? align256((size_t)p.q_start[p.B] * p.H * 2 * sizeof(float)) : 0);
    s.bytes = s.scores + (weights ? (size_t)scores * sizeof(float) : 0);
    return s;
}

}  // namespace

size_t zt_attn_paged_workspace(const int *q_start, const int *n_rows, int B, int n_heads, int n_kv_heads, int dim,
                               int weights) {
    if (B < 1 || !zt_attn_dim_ok(dim) || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 ||
        n_heads > 65535 || !q_start || !n_rows || q_start[0] < 0)
        return 0;
    for (int b = 0; b < B; ++b) {
        const long long q_len = (long long)q_start[b + 1] - q_start[b];
        if (n_rows[b] < 0 || q_len < 0 || q_len > n_rows[b] || q_len * n_heads > INT32_MAX) return 0;
    }
    return paged_space(paged_plan(q_start, n_rows, B, n_heads, n_kv_heads, dim), weights != 0).bytes;
}

int zt_attn_paged(const float *q, const float *k_pages, const float *v_pages, const int *table, float *out, float *lse,
                  const float *w_in, float *w_out, const int *q_start, const int *n_rows, int B, int n_pages,
                  int page_size, int table_stride, int w_stride, int n_heads, int n_kv_heads, int dim, void *workspace,
                  size_t workspace_bytes, hipStream_t stream) {
    if (paged_check("attn_paged", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_heads, n_kv_heads)) return 1;
    if (paged_tokens_check("attn_paged", q_start, n_rows, B, n_heads)) return 1;
    if (!w_in != !w_out) {
        fprintf(stderr, "zt_attn: attn_paged takes w_in and w_out together or neither.\n");
        return 1;
    }
    const bool weights = w_out != nullptr;
    if (weights && paged_weights_check("attn_paged", n_rows, B, w_stride)) return 1;
    const PagedPlan p = paged_plan(q_start, n_rows, B, n_heads, n_kv_heads, dim);
    const PagedSpace space = paged_space(p, weights);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes)) {
        fprintf(stderr, "zt_attn: attn_paged workspace of %zu bytes is short of the %zu needed.\n", workspace_bytes,
                space.bytes);
        return 1;
    }
    if (space.bytes && !workspace_aligned(workspace, "attn_paged")) return 1;
    if (!k_pages || !v_pages || !table || (q_start[B] > q_start[0] && (!q || !out))) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {q, k_pages, v_pages, out})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;

    char *const ws = static_cast<char *>(workspace);
    const int dp = paged_dp(dim);
    PagedArgs a{};
    a.pool = page_pool(const_cast<float *>(k_pages), const_cast<float *>(v_pages), table, n_pages, page_size,
                       table_stride);
    a.q = q; a.out = out; a.lse = lse;
    a.part_acc = reinterpret_cast<float *>(ws);
    a.part_ml = reinterpret_cast<float *>(ws + space.ml);
    a.stat = weights ? reinterpret_cast<float *>(ws + space.stat) : nullptr;
    a.H = n_heads; a.Hkv = n_kv_heads; a.G = p.G; a.dim = dim;
    a.part_ld = p.part_ld;
    a.scale_log2e = (float)(1.4426950408889634 / std::sqrt((double)dim));
    // Whole 16-byte chunks throughout a row.
    const char *const any = dim == dp ? "" : "_any";

    // Launches `name` for the sequences that `items` has work items for, up to ZT_PAGED_MAXB at a time; per_wg items
    // to a workgroup.  `each` fills in argument block x's entry i for sequence b.
    const auto launch_for = [&](const char *name, unsigned threads, unsigned per_wg, auto &x, auto items, auto each) -> int {
        long long blocks = 0;
        x.ns = 0;
        const auto flush = [&]() -> int {
            const unsigned long long wgs = ((unsigned long long)blocks + per_wg - 1) / per_wg;
            const bool bad = x.ns && (!grid_ok(wgs, threads) || launch(st, name, (unsigned)wgs, x, stream, threads));
            x.ns = 0;
            blocks = 0;
            return bad;
        };
        for (int b = 0; b < B; ++b) {
            const long long n = items(b);
            if (n > 0) {
                if ((x.ns == ZT_PAGED_MAXB || blocks + n > INT32_MAX) && flush()) return 1;
                if (n > INT32_MAX) {
                    grid_ok((unsigned long long)n, threads);  // says why
                    return 1;
                }
                const int i = x.ns++;
                x.b[i] = b; x.q0[i] = q_start[b]; x.q_len[i] = p.q_len(b); x.n_rows[i] = n_rows[b];
                x.first[i] = (int)blocks;
                each(i, b);
                blocks += n;
            }
            each(-1, b);  // after it
        }
        return flush();
    };
    char name[64];
    for (const PagedKind kind : kPagedKinds) {
        const bool many = kind == PagedKind::Many;
        a.chunk = many ? p.chunk_many : p.chunk_few;
        a.scores = weights && !many ? reinterpret_cast<float *>(ws + space.scores) : nullptr;
        long long part0 = 0, score0 = 0;
        const auto fill = [&](int i, int b) {
            if (i < 0) {
                part0 += p.slots(b);
                score0 += p.scores(b);
                return;
            }
            a.nch[i] = p.chunks(b);
            a.part0[i] = part0;
            a.score0[i] = score0;
        };
        const auto mine = [&](int b) { return p.kind(b) == kind; };
        if (many) snprintf(name, sizeof name, "zt_paged_many_d%d_8%d%s", dp, dp <= 128 ? 2 : 1, any);
        else snprintf(name, sizeof name, "zt_paged_few_d%d_n%d%s", dp, kind == PagedKind::Few1 ? 1 : 2, any);
        if (launch_for(name, many ? 512u : 256u, 1, a, [&](int b) { return mine(b) ? p.items(b) : 0LL; }, fill)) return 1;
        // Same stream: the merge reads the chunks' partials.
        part0 = score0 = 0;
        snprintf(name, sizeof name, "zt_paged_merge_d%d", dp);
        const auto merged = [&](int b) { return mine(b) && p.chunks(b) > 1 ? (long long)p.q_len(b) * n_heads : 0LL; };
        if (launch_for(name, 256u, 4, a, merged, fill)) return 1;
    }
    if (!weights) return 0;
    // ... and these the rows' statistics.
    PagedWeightArgs g{};
    g.pool = a.pool; g.q = q; g.stat = a.stat; g.w_in = w_in; g.w_out = w_out;
    g.scores = g.parts = reinterpret_cast<float *>(ws + space.scores);
    g.H = n_heads; g.Hkv = n_kv_heads; g.G = p.G; g.dim = dim; g.w_stride = w_stride;
    g.part_rows = p.part_rows;
    g.scale_log2e = a.scale_log2e;
    long long score0 = 0;
    const auto fill = [&](int i, int b) {
        if (i < 0) score0 += p.scores(b);
        else g.score0[i] = score0;
    };
    const auto per_head = [&](int b, int keys) { return (long long)((n_rows[b] + keys - 1) / keys) * n_kv_heads; };
    if (launch_for("zt_paged_weights", 256u, 1, g, [&](int b) { return p.many(b) ? 0LL : per_head(b, 1024); }, fill)) return 1;
    score0 = 0;
    snprintf(name, sizeof name, "zt_paged_wparts_d%d%s", dp, any);
    const auto parts = [&](int b) { return p.many(b) ? per_head(b, p.weight_keys()) * p.parts(b) : 0LL; };
    if (launch_for(name, 512u, 1, g, parts, fill)) return 1;
    score0 = 0;
    snprintf(name, sizeof name, "zt_paged_wsum_%d", p.weight_keys());
    return launch_for(name, 256u, 1, g, [&](int b) { return p.many(b) ? per_head(b, 256) : 0LL; }, fill);
}

int zt_paged_append(const float *q, const float *k_new, const float *v_new, float *q_out, float *k_pages, float *v_pages,
                    const int *table, float *w, const int *q_start, const int *n_rows, const int *pos, int B, int n_pages,
                    int page_size, int table_stride, int w_stride, int n_heads, int n_kv_heads, int dim, double theta,
                    hipStream_t stream) {
    if (paged_check("paged_append", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_heads, n_kv_heads)) return 1;
    if (paged_tokens_check("paged_append", q_start, n_rows, B, n_heads)) return 1;
    if (w && paged_weights_check("paged_append", n_rows, B, w_stride)) return 1;
    if (!pos) {
        fprintf(stderr, "zt_attn: paged_append needs the host pos array.\n");
        return 1;
    }
    for (int b = 0; b < B; ++b) {
        if (pos[b] < 0 || (long long)pos[b] + (q_start[b + 1] - q_start[b]) > INT32_MAX) {
            fprintf(stderr, "zt_attn: sequence %d appends at position %d.\n", b, pos[b]);
            return 1;
        }
    }
    if (!(theta > 0.0)) {
        fprintf(stderr, "zt_attn: RoPE theta %g is not usable.\n", theta);
        return 1;
    }
    const bool any = q_start[B] > q_start[0];
    if (!k_pages || !v_pages || !table || (any && (!k_new || !v_new)) || !q != !q_out) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {q, k_new, v_new, q_out, k_pages, v_pages})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;
    PagedAppendArgs a{};
    a.pool = page_pool(k_pages, v_pages, table, n_pages, page_size, table_stride);
    a.q = q; a.k_new = k_new; a.v_new = v_new; a.q_out = q_out; a.w = w;
    a.H = n_heads; a.Hkv = n_kv_heads; a.dim = dim; a.w_stride = w_stride; a.theta = theta;
    const int per = std::min(16, 256 / (dim / 2));  // tokens of a workgroup
    const long long tasks = ((q ? n_heads : 0) + 2LL * n_kv_heads) * (dim / 2);
    for (int b = 0; b < B;) {
        a.ns = 0;
        a.token0 = q_start[b];
        for (; b < B && a.ns < ZT_PAGED_MAXB; ++b) {
            const int q_len = q_start[b + 1] - q_start[b];
            if (q_len == 0) continue;
            const int i = a.ns++;
            a.b[i] = b; a.q0[i] = q_start[b]; a.row0[i] = n_rows[b] - q_len; a.pos[i] = pos[b];
        }
        a.tokens = q_start[b] - a.token0;
        if (a.tokens == 0) continue;
        const long long groups = (a.tokens + per - 1) / per;
        a.slices = (int)std::max(1LL, std::min(512 / groups, (std::min(a.tokens, per) * tasks + kThreads - 1) / kThreads));
        if (!grid_ok((unsigned long long)groups * a.slices)) return 1;
        if (launch(st, "zt_rope_paged", (unsigned)(groups * a.slices), a, stream)) return 1;
    }
    return 0;
}

int zt_paged_evict(float *k_pages, float *v_pages, const int *table, const int *table_out, const float *w_in,
                   float *w_out, int *kept, const int *n_rows, int B, int n_pages, int page_size, int table_stride,
                   int w_stride, int n_kv_heads, int dim, int n_first, int n_last, int budget, hipStream_t stream) {
    if (paged_check("paged_evict", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_kv_heads, n_kv_heads)) return 1;
    if (n_first < 0 || n_last < 0 || budget < 1 || n_first > budget - n_last) {
        fprintf(stderr, "zt_attn: a budget of %d rows with the first %d and the last %d kept is not usable.\n", budget,
                n_first, n_last);
        return 1;
    }
    if (paged_weights_check("paged_evict", n_rows, B, w_stride)) return 1;
    if (!k_pages || !v_pages || !table || !table_out || !w_in || !w_out || !kept) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (!rows_aligned(dim, {k_pages, v_pages})) return 1;
    DeviceState *st = require_device();
    if (!st) return 1;
    PagedEvictArgs a{};
    a.pool = page_pool(k_pages, v_pages, table, n_pages, page_size, table_stride);
    a.table_out = table_out; a.w_in = w_in; a.w_out = w_out; a.kept = kept;
    a.Hkv = n_kv_heads; a.dim = dim; a.w_stride = w_stride;
    a.n_first = n_first; a.n_last = n_last; a.budget = budget;
    const int n = dim % 4 == 0 ? 4 : 2, per_head = dim / n;
    for (int b0 = 0; b0 < B; b0 += ZT_PAGED_MAXB) {
        a.b0 = b0;
        a.ns = std::min(B - b0, ZT_PAGED_MAXB);
        int most = 0;
        for (int i = 0; i < a.ns; ++i) {
            a.n_rows[i] = n_rows[b0 + i];
            most = std::max(most, a.n_rows[i]);
        }
        if (!grid_ok((unsigned long long)a.ns * n_kv_heads, 1024)) return 1;
        if (launch(st, "zt_evict_select", (unsigned)(a.ns * n_kv_heads), a, stream, 1024)) return 1;
        // Same stream: the rows move as `kept` says.
        if (table_out == table) {
            if (most <= budget) continue;
            const unsigned long long waves = (unsigned long long)a.ns * n_kv_heads * 2 * ((per_head + 7) / 8);
            if (!grid_ok((waves + 3) / 4)) return 1;
            if (launch(st, n == 4 ? "zt_evict_move_4" : "zt_evict_move_2", (unsigned)((waves + 3) / 4), a, stream))
                return 1;
        } else {
            const int rows_per_wg = std::max(1, 1024 / (n_kv_heads * per_head));
            const unsigned long long blocks = (unsigned long long)a.ns * ((budget + rows_per_wg - 1) / rows_per_wg);
            if (!grid_ok(blocks)) return 1;
            if (launch(st, n == 4 ? "zt_evict_copy_4" : "zt_evict_copy_2", (unsigned)blocks, a, stream)) return 1;
        }
    }
    return 0;
}
