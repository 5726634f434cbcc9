// Pages of a paged cache (gfx950): forking and growing sequences, freeing, compacting the pool, copying pages, and
// moving the rows that a tree of drafted tokens leaves.
//
// refs[p] counts the page-table entries that name page p; a page is free where it is 0.  What a call takes follows
// from the tables and the counts alone, whatever the order its workgroups run in: free pages are taken from the lowest
// number up, so the same state gives the same tables.  Counts change by atomic additions only, whose order does not
// matter.
#include "common.h"
#include "args.h"
#include "paged.h"

DEVI bool is_page(int p, int n_pages) { return (unsigned)p < (unsigned)n_pages; }

// Sum over the threads below (exclusive), and over all of a workgroup's; a uniform call of the whole workgroup.
template <int NW>
DEVI int block_scan(int x, int *total, int (&waves)[NW]) {
    const int lane = lane_id(), w = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(s, d, 64);
        if (lane >= d) s += y;
    }
    __syncthreads();  // the last call's reads
    if (lane == 63) waves[w] = s;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        before += i < w ? waves[i] : 0;
        all += waves[i];
    }
    *total = all;
    return before + s - x;
}

// Sum of counts[0 .. n), by a whole workgroup.
DEVI int block_sum(const int *counts, int n, int (&waves)[4]) {
    int x = 0, total;
    for (int i = threadIdx.x; i < n; i += 256) x += counts[i];
    block_scan(x, &total, waves);
    return total;
}

// The pages of a pool that one workgroup of 1024 threads numbers: thread t takes pages 1024 e + t.  before[e]: how many
// pages before the thread's e-th one have flag(e); returned: how many have it at all.
struct OnePool {
    static constexpr int E = ZT_PAGES_ONE / 1024;
    int counts[E * 16];  // of each 64 pages, then before them
};
template <class Flag>
DEVI int pool_number(OnePool &s, Flag flag, int (&before)[OnePool::E], int (&waves)[16]) {
    constexpr int E = OnePool::E;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const unsigned long long m = __builtin_amdgcn_ballot_w64(flag(e));
        before[e] = __popcll(m & ((1ull << lane) - 1));
        if (lane == 0) s.counts[16 * e + w] = __popcll(m);
    }
    __syncthreads();
    const int x = tid < 16 * E ? s.counts[tid] : 0;
    int total;
    const int at = block_scan(x, &total, waves);
    if (tid < 16 * E) s.counts[tid] = at;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) before[e] += s.counts[16 * e + w];
    return total;
}

// ---- Fork and growth --------------------------------------------------------------------
//
// Entry i: sequence dst goes on from src's first n_rows rows, with pages for n_room.  Of its table's columns those
// below whole = n_rows / page are src's pages (one reference more each, where dst is another sequence); the columns
// from there to want = ceil(n_room / page) are its own: kept where src is dst and nobody else refers to the page, else
// fresh ones.  A fresh page for column `whole` of a partly filled one is asked to be copied: pairs[i].
// Three launches: (1) the free pages of each segment, and each entry's fresh columns, are counted; (2) the free pages
// are numbered and listed, as many as could be wanted; (3) each entry takes those of its numbers.  If there are too
// few, nothing is changed but `missing`.  Few columns in a pool of up to ZT_PAGES_ONE pages: zt_pool_fork_one.
// Bound: a launch, and in it a chain of trips to memory (arguments, table, counts); an entry's pages are all in flight.
extern "C" __global__ void __launch_bounds__(256) zt_pool_count(ForkArgs a) {
    __shared__ int waves[4];
    if ((int)blockIdx.x >= a.n) {  // a segment
        const int seg = (int)blockIdx.x - a.n, p0 = seg * a.segment, len = min(a.segment, a.n_pages - p0);
        int x = 0, total;
        for (int i = threadIdx.x; i < len; i += 256) x += a.refs[p0 + i] == 0;
        block_scan(x, &total, waves);
        if (threadIdx.x == 0) a.seg_free[seg] = total;
        return;
    }
    const int i = blockIdx.x, whole = a.n_rows[i] >> a.shift, want = (a.n_room[i] + (1 << a.shift) - 1) >> a.shift;
    const int *row = a.table + (size_t)a.src[i] * a.table_stride;
    int *rank = a.rank + a.slot0[i];
    int fresh = 0;
    if (a.src[i] != a.dst[i]) {
        fresh = max(0, want - whole);  // all of them
    } else {
        for (int j0 = whole; j0 < want; j0 += 256) {
            const int j = j0 + (int)threadIdx.x;
            bool take = false;
            if (j < want) {
                const int p = row[j];
                take = !(is_page(p, a.n_pages) && a.refs[p] == 1);
            }
            int total;
            const int before = block_scan(take, &total, waves);
            if (j < want) rank[j - whole] = take ? fresh + before : -1;
            fresh += total;
        }
    }
    if (threadIdx.x == 0) a.entry_fresh[a.entry0 + i] = fresh;
}

extern "C" __global__ void __launch_bounds__(256) zt_pool_list(ForkArgs a) {
    __shared__ int waves[4];
    const int seg = blockIdx.x, p0 = seg * a.segment, len = min(a.segment, a.n_pages - p0);
    int at = block_sum(a.seg_free, seg, waves);
    for (int i0 = 0; i0 < len && at < a.slots; i0 += 256) {  // workgroup-uniform
        const int i = i0 + (int)threadIdx.x;
        const bool free = i < len && a.refs[p0 + i] == 0;
        int total;
        const int k = at + block_scan(free, &total, waves);
        if (free && k < a.slots) a.list[k] = p0 + i;
        at += total;
    }
}

extern "C" __global__ void __launch_bounds__(256) zt_pool_fork(ForkArgs a) {
    __shared__ int waves[4];
    const int i = blockIdx.x, src = a.src[i], dst = a.dst[i];
    const int whole = a.n_rows[i] >> a.shift, want = (a.n_room[i] + (1 << a.shift) - 1) >> a.shift;
    const bool self = src == dst, part = (a.n_rows[i] & ((1 << a.shift) - 1)) != 0;
    const int free = block_sum(a.seg_free, a.segments, waves);
    const int before = block_sum(a.entry_fresh, a.entry0 + i, waves);
    const int behind = block_sum(a.entry_fresh + a.entry0 + i, a.entries - a.entry0 - i, waves);
    const int short_of = before + behind - free;
    if (threadIdx.x == 0) {
        if (a.entry0 + i == 0) *a.missing = max(0, short_of);
        a.pairs[2 * i] = a.pairs[2 * i + 1] = -1;
    }
    if (short_of > 0) return;  // workgroup-uniform
    __syncthreads();           // the pair's -1 before its pages
    const int *from = a.table + (size_t)src * a.table_stride;
    int *to = a.table + (size_t)dst * a.table_stride;
    for (int j = (self ? whole : 0) + (int)threadIdx.x; j < want; j += 256) {
        const int p = from[j];
        const bool there = is_page(p, a.n_pages);
        if (j < whole) {
            to[j] = p;
            if (there) atomicAdd(a.refs + p, 1);
            continue;
        }
        const int k = self ? a.rank[a.slot0[i] + j - whole] : j - whole;
        if (k < 0) continue;
        const int f = a.list[before + k];
        to[j] = f;
        atomicAdd(a.refs + f, 1);
        if (self && there) atomicSub(a.refs + p, 1);
        if (j == whole && part) {
            a.pairs[2 * i] = p;
            a.pairs[2 * i + 1] = f;
        }
    }
    if (!self)  // behind its pages a new sequence has none (64 bits: the step past a wide table's end is one past an int's)
        for (long long j = want + (int)threadIdx.x; j < a.table_stride; j += 256) to[j] = -1;
}

// The same by one workgroup, a wave to an entry.  The entries are read from the arguments, which are far, once, all at
// the same time.
extern "C" __global__ void __launch_bounds__(1024) zt_pool_fork_one(ForkArgs a) {
    constexpr int E = OnePool::E;
    struct Entry {
        int src, dst, whole, want, part, slot0;
    };
    __shared__ Entry entry[ZT_PAGES_MAXE];
    __shared__ int waves[16], base[ZT_PAGES_MAXE];
    __shared__ int rank[ZT_PAGES_ONE_SLOTS], list[ZT_PAGES_ONE_SLOTS];
    __shared__ OnePool pool;
    const int tid = threadIdx.x, lane = tid & 63, page = 1 << a.shift;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The thread's pages, loaded now, used below.
    int mine[E];
#pragma unroll
    for (int e = 0; e < E; ++e) mine[e] = 1024 * e + tid < a.n_pages ? a.refs[1024 * e + tid] : 1;
    if (tid < a.n) {
        const int rows = a.n_rows[tid], room = a.n_room[tid];
        entry[tid] = {a.src[tid], a.dst[tid], rows >> a.shift, (room + page - 1) >> a.shift, rows & (page - 1), a.slot0[tid]};
    }
    __syncthreads();
    for (int i = w; i < a.n; i += 16) {
        const Entry x = entry[i];
        int fresh = 0;
        if (x.src != x.dst) {
            fresh = x.want - x.whole;
        } else {
            const int *row = a.table + (size_t)x.src * a.table_stride;
            for (int j0 = x.whole; j0 < x.want; j0 += 64) {  // wave-uniform
                const int j = j0 + lane;
                bool take = false;
                if (j < x.want) {
                    const int p = row[j];
                    take = !(is_page(p, a.n_pages) && a.refs[p] == 1);
                }
                const unsigned long long all = __builtin_amdgcn_ballot_w64(take);
                if (j < x.want) rank[x.slot0 + j - x.whole] = take ? fresh + __popcll(all & ((1ull << lane) - 1)) : -1;
                fresh += __popcll(all);
            }
        }
        if (lane == 0) base[i] = fresh;
    }
    int before[E];
    const int total = pool_number(pool, [&](int e) { return mine[e] == 0; }, before, waves);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (mine[e] == 0 && before[e] < a.slots) list[before[e]] = 1024 * e + tid;
    // Every thread has read what it needs of the counts: they may change from here on.
    const int x = tid < a.n ? base[tid] : 0;  // (written before the numbering's barriers)
    int fresh;
    const int first = block_scan(x, &fresh, waves);
    if (tid < a.n) base[tid] = first;
    if (tid == 0) *a.missing = max(0, fresh - total);
    for (int i = tid; i < 2 * a.n; i += 1024) a.pairs[i] = -1;
    __syncthreads();
    if (fresh > total) return;  // workgroup-uniform
    const auto put = [&](int i, const Entry &x, int j, int p) {  // column j of entry i, where its source has p
        const bool self = x.src == x.dst, there = is_page(p, a.n_pages);
        int *to = a.table + (size_t)x.dst * a.table_stride + j;
        if (j >= x.want) {
            if (!self) *to = -1;
        } else if (j < x.whole) {
            if (self) return;
            *to = p;
            if (there) atomicAdd(a.refs + p, 1);
        } else {
            const int r = self ? rank[x.slot0 + j - x.whole] : j - x.whole;
            if (r < 0) return;
            const int f = list[base[i] + r];
            *to = f;
            atomicAdd(a.refs + f, 1);
            if (self && there) atomicSub(a.refs + p, 1);
            if (j == x.whole && x.part) {
                a.pairs[2 * i] = p;
                a.pairs[2 * i + 1] = f;
            }
        }
    };
    // 64 columns of an entry at a time, of one that grows only those that it may change, and four such pieces: their
    // reads do not wait for one another.
    constexpr int U = 4;
    const int items = a.n * a.pieces;
    for (int item0 = w; item0 < items; item0 += 16 * U) {
        int p[U], at[U];  // at: the column, or -1
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int item = min(item0 + 16 * u, items - 1), i = item / a.pieces;
            const Entry x = entry[i];
            const bool self = x.src == x.dst;
            const int j = (self ? x.whole : 0) + (item - i * a.pieces) * 64 + lane;
            at[u] = item0 + 16 * u < items && j < (self ? x.want : a.table_stride) ? j : -1;
            p[u] = at[u] >= 0 ? a.table[(size_t)x.src * a.table_stride + j] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(item0 + 16 * u, items - 1) / a.pieces;
            if (at[u] >= 0) put(i, entry[i], at[u], p[u]);
        }
    }
}

// ---- Freeing ------------------------------------------------------------------------------
//
// Sequence b keeps its table's first from[i] pages; the entries behind them lose their reference and become -1.
extern "C" __global__ void __launch_bounds__(256) zt_pool_free(FreeArgs a) {
    const int i = (int)blockIdx.x / a.blocks;
    const long long j = a.from[i] + (long long)((int)blockIdx.x % a.blocks) * 256 + threadIdx.x;
    if (j >= a.table_stride) return;
    int *at = a.table + (size_t)a.b[i] * a.table_stride + j;
    const int p = *at;
    if (p == -1) return;
    *at = -1;
    if (is_page(p, a.n_pages)) atomicSub(a.refs + p, 1);
}

// ---- Compaction ----------------------------------------------------------------------------
//
// With L pages in use: the k-th lowest free page below L takes what the k-th highest page in use, past L, holds (there
// are as many of the one as of the other), for k < max_pairs.  For small tables and up to ZT_PAGES_ONE pages a workgroup
// does it by itself (zt_pool_compact_one); else in three launches: (1) the pages in use of each segment are counted; (2)
// both kinds are numbered: pairs, and of each page what becomes of it; (3) tables and counts are written.
constexpr int kStays = -1, kFilled = -2;  // else the number of the pair that it is the source of

extern "C" __global__ void __launch_bounds__(256) zt_pool_used(CompactArgs a) {
    __shared__ int waves[4];
    const long long step = 256LL * gridDim.x;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < 2LL * a.max_pairs; i += step) a.pairs[i] = -1;
    const int seg = blockIdx.x, p0 = seg * a.segment, len = min(a.segment, a.n_pages - p0);
    int x = 0, total;
    for (int i = threadIdx.x; i < len; i += 256) x += a.refs[p0 + i] != 0;
    block_scan(x, &total, waves);
    if (threadIdx.x == 0) a.seg_used[seg] = total;
}

extern "C" __global__ void __launch_bounds__(256) zt_pool_pair(CompactArgs a) {
    __shared__ int waves[4];
    const int seg = blockIdx.x, p0 = seg * a.segment, len = min(a.segment, a.n_pages - p0);
    int used = block_sum(a.seg_used, seg, waves);  // below the segment
    const int L = used + block_sum(a.seg_used + seg, a.segments - seg, waves);
    if (L == a.n_pages && seg == 0 && threadIdx.x == 0) a.moved[0] = a.moved[1] = 0;
    for (int i0 = 0; i0 < len; i0 += 256) {  // workgroup-uniform
        const int i = i0 + (int)threadIdx.x, p = i < len ? p0 + i : 0;
        const bool live = i < len && a.refs[p] != 0;
        int total;
        const int before = used + block_scan(live, &total, waves);  // in use below p
        used += total;
        if (i >= len) continue;
        int becomes = kStays;
        if (live && p >= L && L - 1 - before < a.max_pairs) {  // from the highest down
            becomes = L - 1 - before;
            a.pairs[2 * (size_t)becomes] = p;
        }
        if (!live && p < L && p - before < a.max_pairs) {  // from the lowest up
            becomes = kFilled;
            a.pairs[2 * (size_t)(p - before) + 1] = p;
        }
        a.becomes[p] = becomes;
        if (p == L) {  // the pages in use from here on
            const int all = L - before, m = min(all, a.max_pairs);
            a.moved[0] = m;
            a.moved[1] = all - m;
        }
    }
}

extern "C" __global__ void __launch_bounds__(256) zt_pool_move(CompactArgs a) {
    const long long step = 256LL * gridDim.x, id = (long long)blockIdx.x * 256 + threadIdx.x;
    for (long long i = id; i < a.entries; i += step) {
        const int p = a.table[i], pair = is_page(p, a.n_pages) ? a.becomes[p] : kStays;
        a.table_out[i] = pair >= 0 ? a.pairs[2 * (size_t)pair + 1] : p;
    }
    // A count goes with its page: the source's thread writes both.
    for (long long p = id; p < a.n_pages; p += step) {
        const int pair = a.becomes[p];
        if (pair == kFilled) continue;
        const int r = a.refs[p];
        if (pair >= 0) a.refs_out[a.pairs[2 * (size_t)pair + 1]] = r;
        if (pair >= 0 || a.refs_out != a.refs) a.refs_out[p] = pair >= 0 ? 0 : r;
    }
}

// The same by one workgroup; the new numbers of all pages are kept in LDS.  Bound: a thread's table entries one after the
// other, each a trip to memory: of 16384 pages and 1024 entries 8.1 us, 12288 10.0, 65536 19.5.
extern "C" __global__ void __launch_bounds__(1024) zt_pool_compact_one(CompactArgs a) {
    constexpr int E = OnePool::E;
    __shared__ int waves[16], holes[ZT_PAGES_ONE / 2], now[ZT_PAGES_ONE], above;
    __shared__ OnePool pool;
    const int tid = threadIdx.x;
    int mine[E], before[E];  // before: pages in use below
#pragma unroll
    for (int e = 0; e < E; ++e) mine[e] = 1024 * e + tid < a.n_pages ? a.refs[1024 * e + tid] : 0;
    if (tid == 0) above = 0;
    const int L = pool_number(pool, [&](int e) { return mine[e] != 0; }, before, waves);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int p = 1024 * e + tid;
        // (A hole below L has a page in use past L to fill it: there are at most half as many as pages.)
        if (p < L && mine[e] == 0 && p - before[e] < a.max_pairs) holes[p - before[e]] = p;
        if (p == L && p < a.n_pages) above = L - before[e];  // pages in use from L on
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int p = 1024 * e + tid;
        if (p >= a.n_pages) break;
        const int k = L - 1 - before[e];  // of a page in use past L, from the highest down
        const bool moves = mine[e] != 0 && p >= L && k < a.max_pairs;
        const bool filled = mine[e] == 0 && p < L && p - before[e] < a.max_pairs;
        int to = p;
        if (moves) {
            to = holes[k];
            a.pairs[2 * (size_t)k] = p;
            a.pairs[2 * (size_t)k + 1] = to;
            a.refs_out[to] = mine[e];
            a.refs_out[p] = 0;
        } else if (!filled && a.refs_out != a.refs) {
            a.refs_out[p] = mine[e];
        }
        now[p] = to;
    }
    __syncthreads();
    const int m = min(above, a.max_pairs);
    if (tid == 0) {
        a.moved[0] = m;
        a.moved[1] = above - m;
    }
    for (long long i = 2LL * m + tid; i < 2LL * a.max_pairs; i += 1024) a.pairs[i] = -1;
    for (long long i = tid; i < a.entries; i += 1024) {
        const int p = a.table[i];
        a.table_out[i] = is_page(p, a.n_pages) ? now[p] : p;
    }
}

// ---- Copies ---------------------------------------------------------------------------------
//
// Pages of K and V from pairs[2 i] to pairs[2 i + 1], a workgroup 256 x U chunks of N floats at a time.  A pair with a
// number that is none of the pool's is passed over.  Bound: HBM: 600 pages of 64 rows of 8 heads at d = 128 anywhere in a
// pool of 3451, 119 us, 5.3 TB/s (a copy of 2 GiB 4.9); from a pool's end to its holes, with 700 pairs passed over, 131
// (U = 4 4 % more, stores past the caches 10 %).
template <int N>
DEVI void pool_copy(const CopyArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    constexpr int U = ZT_PAGES_COPY / 256;
    const long long items = 2LL * a.n_pairs * a.pieces;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int piece = (int)(item % a.pieces);
        const long long rest = item / a.pieces;
        const int from = a.pairs[2 * (rest >> 1)], to = a.pairs[2 * (rest >> 1) + 1];
        if (!is_page(from, a.n_pages) || !is_page(to, a.n_pages)) continue;
        float *const base = rest & 1 ? a.v : a.k;
        const vec *x = reinterpret_cast<const vec *>(base + (size_t)from * a.page_floats);
        vec *y = reinterpret_cast<vec *>(base + (size_t)to * a.page_floats);
        const long long n = a.page_floats / N, c0 = piece * (long long)ZT_PAGES_COPY + threadIdx.x;
        vec t[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + 256 * u < n) t[u] = __builtin_nontemporal_load(x + c0 + 256 * u);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + 256 * u < n) y[c0 + 256 * u] = t[u];
    }
}
extern "C" __global__ void __launch_bounds__(256) zt_pool_copy_4(CopyArgs a) { pool_copy<4>(a); }
extern "C" __global__ void __launch_bounds__(256) zt_pool_copy_2(CopyArgs a) { pool_copy<2>(a); }

// Rows that stay of a tree of new tokens: new row path[i] becomes new row i, for i < count.  A thread moves N columns
// of K or of V of all of a sequence's rows, eight at a time, read before they are written: a row is overwritten in the step
// of its own number, at the latest when it is read (path[i] >= i), so that each thread's order of steps is enough.
template <int N>
DEVI void pool_keep(const KeepArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    constexpr int U = 8;
    const int s = (int)blockIdx.x / a.blocks, c = ((int)blockIdx.x % a.blocks) * 256 + (int)threadIdx.x;
    const int cols = a.Hkv * (a.dim / N);
    if (c >= 2 * cols) return;
    const int q_len = a.q_len[s], row0 = a.row0[s], n = min(a.count[a.b[s]], q_len);
    const int *path = a.path + a.q0[s], *table = a.pool.table + (size_t)a.b[s] * a.pool.table_stride;
    vec *base = reinterpret_cast<vec *>(c < cols ? a.pool.k : a.pool.v) + (c < cols ? c : c - cols);
    for (int i0 = 0; i0 < n; i0 += U) {
        vec x[U];
        int to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u, p = i < n ? path[i] : -1;
            to[u] = -1;
            if (p <= i || p >= q_len) continue;  // stays, or is no row that may come here
            const int from = pool_row(a.pool, table, row0 + p);
            if (from < 0) continue;
            to[u] = pool_row(a.pool, table, row0 + i);
            x[u] = base[(size_t)from * cols];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (to[u] >= 0) base[(size_t)to[u] * cols] = x[u];
    }
}
extern "C" __global__ void __launch_bounds__(256) zt_pool_keep_4(KeepArgs a) { pool_keep<4>(a); }
extern "C" __global__ void __launch_bounds__(256) zt_pool_keep_2(KeepArgs a) { pool_keep<2>(a); }
