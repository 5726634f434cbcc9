// Entry points of the paged KV cache (include/zt_attn.h): included by zt_attn.cpp
// inside its extern "C" block, whose launcher, checks and device state they use.
//
// The plan of a call -- which kernel takes which sequence, in how many key chunks --
// follows from the host's lengths alone, so that a workspace's size does not depend
// on the device.

// Rows of a sequence, tokens x heads of one, rows of a budget: no sum of two overflows an int.
constexpr long long kPagedMost = 1LL << 30;

// The tokens x heads that one call attends with: over as many rows as a sequence has, every row's scores are still
// counted in 64 bits.
static bool paged_batch_ok(const int *q_start, int B, int n_heads) {
    return ((long long)q_start[B] - q_start[0]) * n_heads <= 2 * kPagedMost;
}

// The cache's geometry; 0 when usable.
static int paged_geometry(const char *who, int B, int n_pages, int page_size, int table_stride) {
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
    return 0;
}

// And its sequences' rows.
static int paged_check(const char *who, const int *n_rows, int B, int n_pages, int page_size, int table_stride) {
    if (paged_geometry(who, B, n_pages, page_size, table_stride)) return 1;
    if (!n_rows) {
        fprintf(stderr, "zt_attn: %s needs the host n_rows array.\n", who);
        return 1;
    }
    const long long most = std::min((long long)table_stride * page_size, kPagedMost);
    for (int b = 0; b < B; ++b) {
        if (n_rows[b] < 0 || n_rows[b] > most) {
            fprintf(stderr, "zt_attn: sequence %d has n_rows %d, outside [0, %lld].\n", b, n_rows[b], most);
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
        if (q_len < 0 || q_len > n_rows[b] || q_len * n_heads > kPagedMost) {
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

// Which kernel takes a sequence, by its rows per kv head (new tokens x heads of the group): the streaming kernel
// with one or two 16-row blocks, or the split-operand one with 64, 128 or 256 rows in a workgroup (past d = 128 64 or
// 128, at d = 256 128: 36 rows of 16 sequences of 2048, 16 over 4 heads, 97 us, in workgroups of 64 106).
enum PagedKind { kFew1, kFew2, kMany64, kMany128, kMany256, kPagedKinds };
constexpr bool paged_few(PagedKind k) { return k <= kFew2; }
// Waves and 16-row blocks per wave of the split-operand kernel.
struct PagedShape {
    int nw, nq;
};
constexpr PagedShape paged_shape(PagedKind k, int dp) {
    return k == kMany64    ? PagedShape{4, 1}
           : k == kMany256 ? PagedShape{8, 2}
           : dp <= 128     ? PagedShape{4, 2}
                           : PagedShape{8, 1};
}

// What a call does for each sequence.
struct PagedPlan {
    const int *q_start, *n_rows;
    int B, H, Hkv, G, dim, dp, part_ld;
    PagedKind as[kPagedKinds];  // the kind whose launch takes each (itself, or a larger one)
    int most[kPagedKinds];      // units of keys (unit()) of a workgroup at most
    int part_rows;              // rows of a part of the weights' sums
    bool keep;                  // the split-operand kernel stores its scores for the weights
    bool two_blocks;            // the streaming kernel takes 17 to 32 rows

    int q_len(int b) const { return q_start[b + 1] - q_start[b]; }
    int rows(int b) const { return q_len(b) * G; }
    bool any(int b) const { return q_len(b) > 0; }
    PagedKind kind(int b) const { return as[kind_of(b)]; }
    PagedKind kind_of(int b) const {
        const int r = rows(b);
        return r <= 16                ? kFew1
               : r <= 32 && two_blocks ? kFew2
               : r <= 64 && dp <= 192 ? kMany64
               : r <= 128 || dp > 128 ? kMany128
                                      : kMany256;
    }
    bool many(int b) const { return any(b) && !paged_few(kind(b)); }
    // Rows of a workgroup, and the keys of its steps: a 16-key tile for each of four waves, or 32.
    int tile_rows(PagedKind k) const {
        return k == kFew1 ? 16 : k == kFew2 ? 32 : 16 * paged_shape(k, dp).nw * paged_shape(k, dp).nq;
    }
    static int unit(PagedKind k) { return paged_few(k) ? 64 : 32; }
    int tiles(int b) const { return (rows(b) + tile_rows(kind(b)) - 1) / tile_rows(kind(b)); }
    // Keys of a chunk: as few chunks as the limit allows, of one length.
    static int chunk_of(int n_rows, int unit, int most) {
        const int steps = (n_rows + unit - 1) / unit, n = (steps + most - 1) / most;
        return (n > 1 ? (steps + n - 1) / n : steps) * unit;
    }
    int chunk(int b) const { return chunk_of(n_rows[b], unit(kind(b)), most[kind(b)]); }
    int chunks(int b) const { return any(b) ? (n_rows[b] + chunk(b) - 1) / chunk(b) : 0; }
    long long items(int b) const { return (long long)tiles(b) * chunks(b) * Hkv; }
    long long slots(int b) const { return chunks(b) > 1 ? (long long)q_len(b) * H * chunks(b) : 0; }
    int kpad(int b) const { return (n_rows[b] + 15) / 16 * 16; }
    // The weights' sums from scores formed again: waves of a workgroup (four, two workgroups to a CU, while LDS has
    // room); and the keys of a workgroup, also of that which reads them.
    int weight_waves() const { return dp <= 192 ? 4 : 8; }
    int weight_keys() const { return keep ? 128 : 16 * weight_waves() * (dp <= 128 ? 2 : 1); }
    int parts(int b) const { return (rows(b) + part_rows - 1) / part_rows; }
    // Floats that the weights need: every row's scores, and the parts' sums.
    long long scores(int b) const {
        if (many(b)) return keep ? (long long)kpad(b) * Hkv * ((rows(b) + 15) / 16 * 16) : 0;
        return (long long)kpad(b) * q_len(b) * H;
    }
    long long sums(int b) const { return many(b) && parts(b) > 1 ? (long long)Hkv * parts(b) * kpad(b) : 0; }
};

// Workgroups of a kind on the device at once, as the plan counts them: of the streaming kernel what the registers of
// one 16-row block allow from d = 64 up (fewer than the 1792 of d = 32; with two blocks 768 stand at d = 64 and 512 at d = 96
// and 128, a quarter to a third less than counted); of the split-operand kernel two of four waves per CU where LDS
// holds both, else one.
int paged_slots(const PagedPlan &p, PagedKind k) {
    if (paged_few(k)) return p.dp <= 64 ? 1024 : p.dp <= 128 ? 768 : p.dp <= 192 ? 512 : 256;
    return paged_shape(k, p.dp).nw == 4 && p.dp <= 192 ? 512 : 256;
}

// When the last workgroup of kind k ends, in steps, were `limit` the most steps of one: the kernel's order of
// items, each to whichever of the device's places (`slots` workgroups) is free first, a workgroup's own
// start and end counted as `extra` steps.  A kv head's items are alike, so that one head's stand for all
// on its share of the places.  *items: how many, all heads.
double paged_span(const PagedPlan &p, PagedKind k, int limit, int slots, double extra, long long *items) {
    const int unit = p.unit(k);
    double busy[512] = {};  // when each place is free, as a heap
    const int places = std::max(1, std::min(512, slots / p.Hkv));
    double end = 0;
    *items = 0;
    for (int b = 0; b < p.B; ++b) {
        if (!p.any(b) || p.kind(b) != k) continue;
        const int c = p.chunk_of(p.n_rows[b], unit, limit) / unit, nt = p.tiles(b);
        const int chunks = ((p.n_rows[b] + unit - 1) / unit + c - 1) / c;
        for (int ci = 0; ci < chunks; ++ci) {
            for (int t = nt - 1; t >= 0; --t) {
                const int last = (std::min(p.rows(b), (t + 1) * p.tile_rows(k)) - 1) / p.G;  // the tile's last token
                const int keys = p.n_rows[b] - p.q_len(b) + last + 1;
                const int left = (keys + unit - 1) / unit - ci * c;
                if (left <= 0) break;  // nor have the tiles before it
                const double at = busy[0] + std::min(left, c) + extra;
                end = std::max(end, at);
                *items += p.Hkv;
                int i = 0;  // the first place takes it and sinks to where it belongs
                for (int j = 1; j < places; j = 2 * i + 1) {
                    if (j + 1 < places && busy[j + 1] < busy[j]) ++j;
                    if (busy[j] >= at) break;
                    busy[i] = busy[j];
                    i = j;
                }
                busy[i] = at;
            }
        }
    }
    return end;
}

// Steps of a workgroup of the split-operand kernel at most.  Keys are cut where whole row tiles would leave CUs
// idle or end unevenly: of the whole and some cuts the one of the least estimated time (paged_span, and the
// partial sums' way to memory and back: 0.011 steps each, a step being RT x 32 keys at 216 TFLOP/s against 4.7 TB/s).
// Measured on MI355X (us, chunks of an even share of all steps / these): 333 tokens on 2340 rows of 32 over 8
// heads at d = 128 139 / 89, a batch with three chunks of 501 on 1850 to 2980 rows at d = 96 513 / 301.
// A workgroup's own start and end count three steps, and a chunk has four at least.  Counted as one or six, eleven of
// twelve shapes take the same time (four sequences of 24 tokens on 2000 rows 46 instead of 53 with either).  With eight
// steps at least 64 tokens on 4096 rows take 58 instead of 46; with two the small grids are 5 to 10 % faster (200 tokens on
// 3000 rows of 8 heads over one 39 / 43) and none of the twelve is slower.
int paged_limit(const PagedPlan &p, PagedKind k, int longest) {
    const int slots = paged_slots(p, k);
    const double extra = 3, way = 0.011;
    const int least = 4;
    int best = longest;
    long long items = 0;
    double time = paged_span(p, k, longest, slots, extra, &items);
    if (items >= 4 * slots) return best;
    int last = longest;
    for (const int cut : {2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128, 192, 256}) {
        const int limit = (longest + cut - 1) / cut;
        if (limit < least || items > 4 * slots) break;
        if (limit == last) continue;
        last = limit;
        const double t = paged_span(p, k, limit, slots, extra, &items) + 1 + way * items;
        if (t < 0.98 * time) {
            time = t;
            best = limit;
        }
    }
    return best;
}

// Units of a workgroup of the streaming kernel at most: the least time by the same reckoning, one unit for a
// workgroup's own start and end.
// Chunks are of one length within a sequence and not over all, so that many workgroups count as an even share
// and half a workgroup besides.  Measured on MI355X (us; 512 / 1024 / 2048 workgroups aimed at / this): 64
// sequences of 4096 to 8192 rows, 32 over 8 heads at d = 128 541 / 572 / 524 / 506, 16 of half that with weights
// 89 / 92 / 88 / 85, 8 of 5200 to 8192 of 8 heads at d = 64 49 / 54 / 49 / 49, one of 100000 rows 158 / 161 / 154 /
// 155.  (Chunks of 64 keys, half of the least: 16 over 4 heads of 8192 rows at d = 256 40 instead of 32.)
int paged_few_limit(const PagedPlan &p, PagedKind k, int longest) {
    const int wgs = tuned(kTunePagedWgs, 0), slots = paged_slots(p, k);
    int best = longest;
    double time = 0;
    for (int limit = 2; limit <= longest; limit += (limit + 3) / 4) {
        long long n = 0, units = 0;
        for (int b = 0; b < p.B; ++b) {
            if (!p.any(b) || p.kind(b) != k) continue;
            const int u = (p.n_rows[b] + 63) / 64;
            n += (u + limit - 1) / limit;
            units += u;
        }
        n *= p.Hkv;
        units *= p.Hkv;
        if (wgs) {  // forced
            if (n <= wgs) return limit;
            continue;
        }
        const double rounds = (double)((n + slots - 1) / slots) * (limit + 1);
        const double t = std::min(rounds, (double)(units + n) / slots + 0.5 * (limit + 1));
        if (limit == 2 || t < time) {
            time = t;
            best = limit;
        }
        if (n <= slots) break;  // fewer workgroups only take longer
    }
    return best;
}

// A kind of few steps joins the next larger kind of the batch, whose empty rows cost less than a launch more (two,
// with a merge), while the workgroups of both are on the device at once and their steps of 32 keys few for each
// place: 7 of the split-operand kernel, 4 of the streaming one.  Measured on MI355X (us, a launch for each /
// joined): every fourth of 12 sequences with 40 new tokens, the others one, 32 over 8 heads at d = 128, 60 rows 26.6
// / 20.9, 200 (2 steps of each place) 46 / 41, 500 (4) 54 / 51; 900, 16 over 4 at d = 256 (7) 68 / 61; 1800 (13) 92
// / 97, at d = 128 82 / 135; 100 sequences of 60 rows (800 workgroups) 36 / 46.  Every fourth of 16 with 6 tokens,
// 500 rows (3) 37 / 28, 900 (5) 44 / 50.
void paged_join(PagedPlan &p) {
    long long wgs[kPagedKinds] = {}, steps[kPagedKinds] = {};
    for (int b = 0; b < p.B; ++b) {
        if (!p.any(b)) continue;
        const long long n = (long long)p.tiles(b) * p.Hkv;
        wgs[p.kind(b)] += n;
        steps[p.kind(b)] += n * ((p.n_rows[b] + 31) / 32);
    }
    for (int k = 0; k + 1 < kPagedKinds; ++k) {
        int larger = k + 1;
        while (larger < kPagedKinds && !wgs[larger]) ++larger;
        if (!wgs[k] || larger == kPagedKinds) continue;
        const int slots = paged_slots(p, (PagedKind)larger);
        if (wgs[k] + wgs[larger] > slots || steps[k] + steps[larger] > (paged_few((PagedKind)larger) ? 4 : 7) * slots)
            continue;
        wgs[larger] += wgs[k];
        steps[larger] += steps[k];
        for (PagedKind &as : p.as)
            if (as == k) as = (PagedKind)larger;
    }
}

PagedPlan paged_plan(const int *q_start, const int *n_rows, int B, int H, int Hkv, int dim) {
    PagedPlan p{q_start, n_rows, B, H, Hkv, H / Hkv, dim, paged_dp(dim), (dim + 3) / 4 * 4, {}, {}, 0, true, true};
    for (int k = 0; k < kPagedKinds; ++k) p.as[k] = (PagedKind)k;
    int longest[kPagedKinds] = {};
    long long scores = 0, sums = 0, units = 0;
    // 17 to 32 rows: with two blocks the streaming kernel's f32 MFMAs weigh as much as its reads, and past d =
    // 128 its registers spill; where that does not hide behind latency the split-operand kernel takes them.
    // Measured on MI355X (us, streaming / split operands; 32 rows): one sequence of 8192 rows of 32 over 8 heads at
    // d = 128 33 / 36, 4 of 500 19.5 / 22.9, 16 of 2048 89 / 70, at d = 96 72 / 66; 16 of 2048 of 12 over 4 heads
    // at d = 64 26 / 27, of 16 over 4 at d = 256 281 / 95.
    for (int b = 0; b < B; ++b)
        if (p.rows(b) > 16 && p.rows(b) <= 32) units += (long long)Hkv * ((n_rows[b] + 63) / 64);
    p.two_blocks = p.dp <= 64 || (p.dp <= 128 && units <= 2048);  // (64 keys a unit: four to each of 512 workgroups)
    paged_join(p);
    for (int b = 0; b < B; ++b) {
        if (!p.any(b)) continue;
        const PagedKind k = p.kind(b);
        longest[k] = std::max(longest[k], (n_rows[b] + p.unit(k) - 1) / p.unit(k));
        if (!paged_few(k)) scores += p.scores(b);
    }
    for (int ki = 0; ki < kPagedKinds; ++ki) {
        const PagedKind k = (PagedKind)ki;
        p.most[k] = !longest[k] ? 1 : paged_few(k) ? paged_few_limit(p, k, longest[k]) : paged_limit(p, k, longest[k]);
    }
    // The split-operand kernel's scores are kept for the weights from d = 64 up while they take no more room than
    // 4 GiB (32 heads of 4096 tokens over 8192 rows), else formed again.  Measured on MI355X (attention and
    // weights, us, kept / again): a prompt of 2048 rows of 32 over 8 heads at d = 128 339 / 388, 64 tokens on 4096
    // rows 66 / 80, 4096 tokens on 8192 rows 2695 / 3048, 2048 rows of 16 over 4 at d = 256 366 / 478, 4 x 1024 of
    // 8 heads at d = 64 96 / 95; 4096 rows of 4 over 2 at d = 32 165 / 143.
    p.keep = tuned(kTunePagedScores, p.dp >= 64 && scores <= 1LL << 30) == 1;
    for (int b = 0; b < B; ++b)
        if (p.many(b)) sums += (long long)p.rows(b) * Hkv * ((n_rows[b] + p.weight_keys() - 1) / p.weight_keys());
    // About 2048 workgroups, of 256 rows at least.
    p.part_rows = (int)std::min(std::max(256LL, (sums / 2048 + 31) / 32 * 32), 1LL << 30);
    return p;
}

// Offsets of a workspace's parts in bytes.
struct PagedSpace {
    size_t ml, stat, scores, sums, bytes;
};
PagedSpace paged_space(const PagedPlan &p, bool weights) {
    long long slots = 0, scores = 0, sums = 0;
    for (int b = 0; b < p.B; ++b) {
        slots += p.slots(b);
        scores += p.scores(b);
        sums += p.sums(b);
    }
    PagedSpace s{};
    s.ml = align256((size_t)slots * p.part_ld * sizeof(float));
    s.stat = s.ml + align256((size_t)slots * 2 * sizeof(float));
    s.scores = s.stat + (weights ? align256((size_t)p.q_start[p.B] * p.H * 2 * sizeof(float)) : 0);
    s.sums = s.scores + (weights ? align256((size_t)scores * sizeof(float)) : 0);
    s.bytes = s.sums + (weights ? (size_t)sums * sizeof(float) : 0);
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
        if (n_rows[b] < 0 || n_rows[b] > kPagedMost || q_len < 0 || q_len > n_rows[b] || q_len * n_heads > kPagedMost) return 0;
    }
    if (!paged_batch_ok(q_start, B, n_heads)) return 0;
    return paged_space(paged_plan(q_start, n_rows, B, n_heads, n_kv_heads, dim), weights != 0).bytes;
}

// New tokens' masks: 64-bit words, one bit per new token of a sequence.
static int tree_words_check(const char *who, const int *q_start, int B, int words) {
    for (int b = 0; b < B; ++b) {
        const int q_len = q_start[b + 1] - q_start[b];
        if (words < 1 || words > (1 << 24) || (long long)words * 64 < q_len) {
            fprintf(stderr, "zt_attn: %s: masks of %d 64-bit words do not hold sequence %d's %d new tokens.\n", who, words,
                    b, q_len);
            return 1;
        }
    }
    return 0;
}

// Attention of a batch's new tokens, with the weights of the rows or without, of a chunk or (mask) of trees.
static int paged_attend(const char *who, const float *q, const float *k_pages, const float *v_pages, const int *table,
                        float *out, float *lse, const float *w_in, float *w_out, const uint64_t *mask, int words,
                        const int *q_start, const int *n_rows, int B, int n_pages, int page_size, int table_stride,
                        int w_stride, int n_heads, int n_kv_heads, int dim, void *workspace, size_t workspace_bytes,
                        bool tree, hipStream_t stream) {
    if (paged_check(who, n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_heads, n_kv_heads)) return 1;
    if (paged_tokens_check(who, q_start, n_rows, B, n_heads)) return 1;
    if (!paged_batch_ok(q_start, B, n_heads)) {
        fprintf(stderr, "zt_attn: %s takes at most %lld new tokens x heads in a call.\n", who, 2 * kPagedMost);
        return 1;
    }
    if (!w_in != !w_out) {
        fprintf(stderr, "zt_attn: %s takes w_in and w_out together or neither.\n", who);
        return 1;
    }
    if (tree && tree_words_check(who, q_start, B, words)) return 1;
    const bool weights = w_out != nullptr;
    if (weights && paged_weights_check(who, n_rows, B, w_stride)) return 1;
    const PagedPlan p = paged_plan(q_start, n_rows, B, n_heads, n_kv_heads, dim);
    const PagedSpace space = paged_space(p, weights);
    if (space.bytes && (!workspace || workspace_bytes < space.bytes)) {
        fprintf(stderr, "zt_attn: %s workspace of %zu bytes is short of the %zu needed.\n", who, workspace_bytes,
                space.bytes);
        return 1;
    }
    if (space.bytes && !workspace_aligned(workspace, who)) return 1;
    if (!k_pages || !v_pages || !table || (q_start[B] > q_start[0] && (!q || !out || (tree && !mask)))) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if (tree && ((uintptr_t)mask & 7)) {
        fprintf(stderr, "zt_attn: masks at %p are not 8-byte aligned.\n", (const void *)mask);
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
    a.w_in = w_in; a.w_out = w_out; a.w_stride = w_stride;
    a.mask = reinterpret_cast<const unsigned *>(mask); a.mask_ld = 2 * words;
    a.scale_log2e = (float)(1.4426950408889634 / std::sqrt((double)dim));
    // Whole 16-byte chunks throughout a row.
    const char *const any = dim == dp ? "" : "_any", *const set = tree ? "tree" : "paged";

    // Launches `name` for the sequences that `items` has work items for, up to ZT_PAGED_MAXB at a time; per_wg items
    // to a workgroup.  `each(i, b)` fills in what else argument block x needs for its entry i, sequence b; each(-1, b)
    // comes behind every sequence.
    const auto launch_for = [&](const char *name, unsigned threads, unsigned per_wg, auto &x, auto items,
                                auto each) -> int {
        const long long most = 0xFFFFFFFFll / threads * per_wg;  // items whose work-items fit a grid
        long long blocks = 0;
        PagedSeqs &s = x.seq;
        s.n = 0;
        const auto flush = [&]() -> int {
            const unsigned long long wgs = ((unsigned long long)blocks + per_wg - 1) / per_wg;
            const bool bad = s.n && (!grid_ok(wgs, threads) || launch(st, name, (unsigned)wgs, x, stream, threads));
            s.n = 0;
            blocks = 0;
            return bad;
        };
        for (int b = 0; b < B; ++b) {
            const long long n = items(b);
            if (n > 0) {
                if ((s.n == ZT_PAGED_MAXB || blocks + n > most) && flush()) return 1;
                if (n > most) return !grid_ok((unsigned long long)n, threads);  // (which says why)
                const int i = s.n++;
                s.b[i] = b; s.q0[i] = q_start[b]; s.q_len[i] = p.q_len(b); s.n_rows[i] = n_rows[b];
                s.first[i] = (int)blocks;
                s.nch[i] = p.chunks(b); s.chunk[i] = p.chunk(b);
                each(i, b);
                blocks += n;
            }
            each(-1, b);  // after it
        }
        return flush();
    };
    char name[64];
    for (int ki = 0; ki < kPagedKinds; ++ki) {
        const PagedKind kind = (PagedKind)ki;
        const bool few = paged_few(kind);
        PagedShape shape = paged_shape(kind, dp);
        // Trees of 65 to 128 rows on a grid of at most one workgroup per CU take eight waves of 16 rows, two to a SIMD, and not
        // four of 32 that nothing runs beside.  Measured on MI355X (us, four / eight): 26 tokens of 32 over 8 heads at d = 128
        // on 1000 rows 31.0 / 24.9, 4103 (208 workgroups) 36.3 / 29.8, 30 of 24 over 8 heads at d = 96 on 4000 27.4 / 24.8, 4
        // sequences of 40 of 12 over 4 at d = 64 on 2000 24.9 / 23.4; past it, 26 on 8000 50.5 / 56.2, two of them 75.5 / 76.0
        // (but 24 sequences of 20 on 3192 to 8114 rows 482.6 / 454.8); 50 of 4 over 2 at d = 32 on 2000 20.3 / 21.5.
        // Chunks stay with the kernels that they had: eight waves of 16 rows are not built for them (26 tokens on 4103 rows
        // as a chunk 36.1).  The shape does not change the plan, whose workspace depends on no device and whose cuts are for
        // two workgroups of four waves to a CU.
        if (tree && kind == kMany128 && dp >= 64 && dp <= 128) {
            long long wgs = 0;
            for (int b = 0; b < B; ++b)
                if (p.any(b) && p.kind(b) == kind) wgs += p.items(b);
            if (wgs <= st->cus) shape = PagedShape{8, 1};
        }
        a.scores = weights && (few || p.keep) ? reinterpret_cast<float *>(ws + space.scores) : nullptr;
        long long part0 = 0, score0 = 0;
        const auto fill = [&](int i, int b) {
            if (i < 0) {
                part0 += p.slots(b);
                score0 += p.scores(b);
                return;
            }
            a.seq.at0[i] = part0;
            a.score0[i] = score0;
        };
        const auto mine = [&](int b) { return p.any(b) && p.kind(b) == kind; };
        if (few) snprintf(name, sizeof name, "zt_%s_few_d%d_n%d%s", set, dp, kind == kFew1 ? 1 : 2, any);
        else snprintf(name, sizeof name, "zt_%s_many_d%d_%d%d%s", set, dp, shape.nw, shape.nq, any);
        const auto items = [&](int b) { return mine(b) ? p.items(b) : 0LL; };
        if (launch_for(name, few ? 256u : 64u * shape.nw, 1, a, items, fill)) return 1;
        // Same stream: the merge reads the chunks' partials.
        part0 = score0 = 0;
        // Many rows of few chunks: a lane group to a row; else a workgroup.
        int chunks = 0;
        for (int b = 0; b < B; ++b)
            if (mine(b)) chunks = std::max(chunks, p.chunks(b));
        if (chunks <= 1) continue;
        const bool by_rows = !few && chunks <= 8;
        // (Few rows' weights come with it, where they are wanted: 1024 keys to a workgroup.)
        const bool with = weights && few;
        snprintf(name, sizeof name,
                 by_rows ? "zt_%s_merge_rows_d%d" : with ? "zt_%s_merge_w_d%d" : "zt_%s_merge_d%d", set, dp);
        const auto merged = [&](int b) {
            const long long sums = with ? (long long)((n_rows[b] + 1023) / 1024) * n_kv_heads : 0;
            return mine(b) && p.chunks(b) > 1 ? (long long)p.q_len(b) * n_heads + sums : 0LL;
        };
        const unsigned per_wg = !by_rows ? 1 : dp <= 32 ? 32 : dp <= 64 ? 16 : dp <= 128 ? 8 : 4;
        if (launch_for(name, 256u, per_wg, a, merged, fill)) return 1;
    }
    if (!weights) return 0;
    // ... and these the rows' statistics.
    PagedWeightArgs g{};
    g.pool = a.pool; g.q = q; g.stat = a.stat; g.w_in = w_in; g.w_out = w_out;
    g.scores = reinterpret_cast<float *>(ws + space.scores);
    g.parts = reinterpret_cast<float *>(ws + space.sums);
    g.H = n_heads; g.Hkv = n_kv_heads; g.G = p.G; g.dim = dim; g.w_stride = w_stride;
    g.part_rows = p.part_rows;
    g.scale_log2e = a.scale_log2e;
    long long score0 = 0, parts0 = 0;
    const auto fill = [&](int i, int b) {
        if (i < 0) {
            score0 += p.scores(b);
            parts0 += p.sums(b);
        } else {
            g.seq.at0[i] = score0;
            g.parts0[i] = parts0;
        }
    };
    const auto run = [&](const char *kernel, unsigned threads, bool many, auto items) {
        score0 = parts0 = 0;
        return launch_for(kernel, threads, 1, g, [&](int b) { return p.many(b) == many ? items(b) : 0LL; }, fill);
    };
    const auto per_head = [&](int b, int keys) { return (long long)((n_rows[b] + keys - 1) / keys) * n_kv_heads; };
    const auto rest = [&](int b) { return p.chunks(b) > 1 ? 0LL : per_head(b, 1024); };  // of those without a merge
    if (run("zt_paged_weights", 256u, false, rest)) return 1;
    if (p.keep) snprintf(name, sizeof name, "zt_paged_wcols");
    else snprintf(name, sizeof name, "zt_paged_wparts_d%d%s", dp, any);
    const auto parts = [&](int b) { return per_head(b, p.weight_keys()) * p.parts(b); };
    if (run(name, p.keep ? 256u : 64u * p.weight_waves(), true, parts)) return 1;
    snprintf(name, sizeof name, "zt_paged_wsum_%d", p.weight_keys());
    return run(name, 256u, true, [&](int b) { return p.parts(b) > 1 ? per_head(b, 256) : 0LL; });
}

int zt_attn_paged(const float *q, const float *k_pages, const float *v_pages, const int *table, float *out, float *lse,
                  const float *w_in, float *w_out, const int *q_start, const int *n_rows, int B, int n_pages,
                  int page_size, int table_stride, int w_stride, int n_heads, int n_kv_heads, int dim, void *workspace,
                  size_t workspace_bytes, hipStream_t stream) {
    return paged_attend("attn_paged", q, k_pages, v_pages, table, out, lse, w_in, w_out, nullptr, 0, q_start, n_rows, B,
                        n_pages, page_size, table_stride, w_stride, n_heads, n_kv_heads, dim, workspace, workspace_bytes,
                        false, stream);
}

int zt_attn_paged_tree(const float *q, const float *k_pages, const float *v_pages, const int *table, const uint64_t *mask,
                       float *out, float *lse, const int *q_start, const int *n_rows, int B, int n_pages, int page_size,
                       int table_stride, int words, int n_heads, int n_kv_heads, int dim, void *workspace,
                       size_t workspace_bytes, hipStream_t stream) {
    return paged_attend("attn_paged_tree", q, k_pages, v_pages, table, out, lse, nullptr, nullptr, mask, words, q_start,
                        n_rows, B, n_pages, page_size, table_stride, 0, n_heads, n_kv_heads, dim, workspace,
                        workspace_bytes, true, stream);
}

int zt_tree_mask(const int *parent, uint64_t *mask, int *pos_out, const int *q_start, const int *pos, int B, int words,
                 hipStream_t stream) {
    if (B < 1 || !q_start || q_start[0] < 0) {
        fprintf(stderr, "zt_attn: tree_mask of %d sequences needs the host q_start array, from 0 up.\n", B);
        return 1;
    }
    for (int b = 0; b < B; ++b) {
        if (q_start[b + 1] < q_start[b]) {
            fprintf(stderr, "zt_attn: sequence %d has %lld new tokens.\n", b, (long long)q_start[b + 1] - q_start[b]);
            return 1;
        }
    }
    if (tree_words_check("tree_mask", q_start, B, words)) return 1;
    if (!pos != !pos_out) {
        fprintf(stderr, "zt_attn: tree_mask takes the host pos array and pos_out together or neither.\n");
        return 1;
    }
    for (int b = 0; pos && b < B; ++b) {
        if (pos[b] < 0 || (long long)pos[b] + (q_start[b + 1] - q_start[b]) > INT32_MAX) {
            fprintf(stderr, "zt_attn: sequence %d's tree begins at position %d.\n", b, pos[b]);
            return 1;
        }
    }
    if (q_start[B] > q_start[0] && (!parent || !mask)) {
        fprintf(stderr, "zt_attn: a null tensor pointer is not launchable.\n");
        return 1;
    }
    if ((uintptr_t)mask & 7) {
        fprintf(stderr, "zt_attn: masks at %p are not 8-byte aligned.\n", (const void *)mask);
        return 1;
    }
    DeviceState *st = require_device();
    if (!st) return 1;
    TreeMaskArgs a{};
    a.parent = parent; a.mask = reinterpret_cast<unsigned long long *>(mask); a.pos = pos_out;
    a.words = words;
    // (The tokens are less than 2^31, 256 to a workgroup: a launch has room for any 64 sequences.)
    for (int b = 0; b < B;) {
        unsigned blocks = 0;
        PagedSeqs &s = a.seq;
        for (s.n = 0; b < B && s.n < ZT_PAGED_MAXB; ++b) {
            const int q_len = q_start[b + 1] - q_start[b];
            if (q_len == 0) continue;
            const int i = s.n++;
            s.b[i] = b; s.q0[i] = q_start[b]; s.q_len[i] = q_len; s.n_rows[i] = pos ? pos[b] : 0;
            s.first[i] = (int)blocks;
            blocks += ((unsigned)q_len + kThreads - 1) / kThreads;
        }
        if (blocks && launch(st, "zt_tree_mask", blocks, a, stream)) return 1;
    }
    return 0;
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
    // Pairs of a thread: both halves of a head in whole chunks of that.
    const int vw = dim % 8 == 0 ? 4 : dim % 4 == 0 ? 2 : 1;
    const long long tasks = ((q ? n_heads : 0) + 2LL * n_kv_heads) * (dim / 2) / vw;
    char name[64];
    snprintf(name, sizeof name, "zt_rope_paged_%d", vw);
    const int most = (int)(0xFFFFFFFFu / kThreads) * per;  // tokens of a launch
    for (int b = 0; b < B;) {
        a.ns = 0;
        const int first = q_start[b];
        for (; b < B && a.ns < ZT_PAGED_MAXB; ++b) {
            const int q_len = q_start[b + 1] - q_start[b];
            if (q_len == 0) continue;
            const int i = a.ns++;
            a.b[i] = b; a.q0[i] = q_start[b]; a.row0[i] = n_rows[b] - q_len; a.pos[i] = pos[b];
        }
        for (long long t = first; t < q_start[b]; t += most) {
            a.token0 = (int)t;
            a.tokens = (int)std::min<long long>(most, q_start[b] - t);
            const long long groups = ((long long)a.tokens + per - 1) / per;
            a.slices = (int)std::max(1LL, std::min(512 / groups, (std::min(a.tokens, per) * tasks + kThreads - 1) / kThreads));
            if (launch(st, name, (unsigned)(groups * a.slices), a, stream)) return 1;
        }
    }
    return 0;
}

int zt_paged_evict(float *k_pages, float *v_pages, const int *table, const int *table_out, const float *w_in,
                   float *w_out, int *kept, const int *n_rows, int B, int n_pages, int page_size, int table_stride,
                   int w_stride, int n_kv_heads, int dim, int n_first, int n_last, int budget, hipStream_t stream) {
    if (paged_check("paged_evict", n_rows, B, n_pages, page_size, table_stride)) return 1;
    if (!zt_attn_dim_ok(dim)) return refuse_dim(dim);
    if (check_group(n_kv_heads, n_kv_heads)) return 1;
    if (n_first < 0 || n_last < 0 || budget < 1 || budget > kPagedMost || n_first > budget - n_last) {
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
    const int n = dim % 4 == 0 ? 4 : 2, per_head = dim / n;
    const bool in_place = table_out == table;
    const char *const move = in_place ? n == 4 ? "zt_evict_move_4" : "zt_evict_move_2"
                                      : n == 4 ? "zt_evict_copy_4" : "zt_evict_copy_2";
    const unsigned move_threads = in_place ? 1024 : kThreads;
    const int rows_per_wg = std::max(1, 1024 / (n_kv_heads * per_head));  // of a copy
    // Workgroups that move a sequence of `most` rows at most: K and V of each head, or its row tiles.
    const auto move_wgs = [&](int most) {
        return in_place ? 2LL * n_kv_heads : ((long long)std::min(budget, most) + rows_per_wg - 1) / rows_per_wg;
    };
    const long long move_most = 0xFFFFFFFFll / move_threads;  // workgroups of a launch
    for (int b = 0; b < B; ++b)
        if (n_rows[b] && move_wgs(n_rows[b]) > move_most) return !grid_ok(move_wgs(n_rows[b]), move_threads);
    DeviceState *st = require_device();
    if (!st) return 1;
    PagedEvictArgs a{};
    a.pool = page_pool(k_pages, v_pages, table, n_pages, page_size, table_stride);
    a.table_out = table_out; a.w_in = w_in; a.w_out = w_out; a.kept = kept;
    a.Hkv = n_kv_heads; a.dim = dim; a.w_stride = w_stride;
    a.n_first = n_first; a.n_last = n_last; a.budget = budget;
    for (int b0 = 0; b0 < B; b0 += ZT_PAGED_MAXB) {
        a.b0 = b0;
        a.ns = std::min(B - b0, ZT_PAGED_MAXB);
        int most = 0;
        for (int i = 0; i < a.ns; ++i) {
            a.n_rows[i] = n_rows[b0 + i];
            most = std::max(most, a.n_rows[i]);
        }
        // By the rows that a workgroup's registers hold.
        const char *select = most <= 1024 ? "zt_evict_select_1024" : most <= 4096 ? "zt_evict_select_4096"
                             : most <= 16384 ? "zt_evict_select_16384" : "zt_evict_select_any";
        const unsigned threads = most <= 1024 ? 256 : most <= 4096 ? 512 : 1024;
        static_assert(ZT_PAGED_MAXB * 65535ull * 1024 <= 0xFFFFFFFFull, "a launch has room for every head's workgroup");
        if (launch(st, select, (unsigned)(a.ns * n_kv_heads), a, stream, threads)) return 1;
        if (in_place ? most <= budget : most == 0) continue;
        // Same stream: the rows move as `kept` says.  As many sequences at a time as a launch has room for, each counted
        // as the longest.
        a.tiles = in_place ? 0 : (int)move_wgs(most);
        const int at_once = (int)std::min<long long>(a.ns, move_most / move_wgs(most));
        for (int i0 = 0, ns = a.ns; i0 < ns; i0 += at_once) {
            a.b0 = b0 + i0;
            a.ns = std::min(ns - i0, at_once);
            for (int i = 0; i < a.ns; ++i) a.n_rows[i] = n_rows[a.b0 + i];
            if (launch(st, move, (unsigned)(a.ns * move_wgs(most)), a, stream, move_threads)) return 1;
        }
    }
    return 0;
}
