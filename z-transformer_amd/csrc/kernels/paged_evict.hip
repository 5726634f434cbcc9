// Eviction from a paged KV cache by accumulated attention weight (gfx950).
//
// A sequence of n rows past its budget keeps, in each kv head by itself, its first n_first
// rows, its last n_last, and of those between the budget - n_first - n_last with the
// largest weight (equal weights: the lower row; NaN below everything).  The kept rows,
// in order of their row, become rows 0 .. budget - 1 of the pages of table_out: the
// same pages (table_out == table) or others.  A sequence within its budget keeps all rows.
#include "args.h"
#include "paged.h"

// Weights as unsigned numbers of the same order: NaN lowest, then -inf .. +inf; -0 is 0.
DEVI unsigned weight_key(float w) {
    if (w != w) return 0;
    const unsigned u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of a wave-uniform count over the workgroup's waves; every thread gets it.
template <int NW>
DEVI int block_count(int mine, int *red) {
    __syncthreads();  // the last reduction's reads
    if (lane_id() == 0) red[threadIdx.x >> 6] = mine;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) s += red[i];
    return s;
}

// Sums of the waves before this one, and of all.
template <int NW>
DEVI int block_before(int mine, int *red, int *all) {
    __syncthreads();
    const int w = threadIdx.x >> 6;
    if (lane_id() == 0) red[w] = mine;
    __syncthreads();
    int before = 0, s = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        before += i < w ? red[i] : 0;
        s += red[i];
    }
    *all = s;
    return before;
}

// Which rows stay: one workgroup of 16 waves per (sequence, kv head).  The threshold, the
// largest key T that at least `need` candidates reach, is found bit by bit from the
// highest; then the rows are walked in order, 1024 at a time, with running counts of those kept and
// of those that equal T.  w may be compacted in place: a block's rows are read before any
// is written, and a row never moves up.
template <int KPT>
DEVI void evict_select(const PagedEvictArgs &a) {
    constexpr int NW = 16;
    __shared__ int red[NW];
    const int tid = threadIdx.x, lane = lane_id();
    const int sl = (int)blockIdx.x / a.Hkv, h = (int)blockIdx.x % a.Hkv, b = a.b0 + sl;
    const int n = a.n_rows[sl];
    const size_t head = (size_t)b * a.Hkv + h;
    const float *w = a.w_in + head * a.w_stride;
    float *wo = a.w_out + head * a.w_stride;
    int *kept = a.kept + head * a.budget;
    if (n <= a.budget) {  // all stay
        for (int i = tid; i < a.budget; i += 64 * NW) kept[i] = i < n ? i : -1;
        if (wo != w)
            for (int i = tid; i < n; i += 64 * NW) wo[i] = w[i];
        return;
    }
    const int lo = a.n_first, hi = n - a.n_last, need = a.budget - a.n_first - a.n_last;
    unsigned T = 0;
    int above = 0;  // candidates past T
    unsigned key[KPT];
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
        const int i = lo + k * 64 * NW + tid;
        key[k] = KPT > 1 && i < hi ? weight_key(w[i]) : 0;
    }
    auto count = [&](unsigned at) {  // candidates whose key is at least `at` (> 0)
        int c = 0;
        if constexpr (KPT > 1) {
#pragma unroll
            for (int k = 0; k < KPT; ++k) c += __popcll(__builtin_amdgcn_ballot_w64(key[k] >= at));
        } else {
            for (int i0 = lo; i0 < hi; i0 += 64 * NW) {
                const int i = i0 + tid;
                c += __popcll(__builtin_amdgcn_ballot_w64(i < hi && weight_key(w[i]) >= at));
            }
        }
        return block_count<NW>(c, red);
    };
    if (need > 0) {
        for (int bit = 31; bit >= 0; --bit) {
            const unsigned trial = T | 1u << bit;
            const int c = count(trial);
            if (c >= need) T = trial;
            else above = c;
        }
    } else {
        T = 0xffffffffu;  // (a NaN's key is 0 and +inf's is less than this: none reaches it)
    }
    const int equal = need - above;  // so many of those that equal T, the lowest rows
    int n_kept = 0, n_equal = 0;
    for (int i0 = 0; i0 < n; i0 += 64 * NW) {
        const int i = i0 + tid;
        const float wi = i < n ? w[i] : 0.f;
        const bool cand = i >= lo && i < hi;
        const unsigned ki = weight_key(wi);
        const unsigned long long eq = __builtin_amdgcn_ballot_w64(cand && ki == T);
        int all_eq = 0;
        const int eq_before = block_before<NW>(__popcll(eq), red, &all_eq) + n_equal;
        const unsigned long long below = (1ull << lane) - 1;
        const bool stay = i < n && (!cand || ki > T || (ki == T && eq_before + __popcll(eq & below) < equal));
        const unsigned long long st = __builtin_amdgcn_ballot_w64(stay);
        int all = 0;
        const int at = block_before<NW>(__popcll(st), red, &all) + n_kept + __popcll(st & below);
        if (stay) {
            kept[at] = i;
            wo[at] = wi;
        }
        n_kept += all;
        n_equal += all_eq;
    }
}

extern "C" __global__ void __launch_bounds__(1024) zt_evict_select(PagedEvictArgs a) { evict_select<1>(a); }

// Rows to other pages: a thread takes 16 (VEC) or 8 bytes of K and V of (row, column).
template <int N>
DEVI void evict_copy(const PagedEvictArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    const int per_head = a.dim / N, per_row = a.Hkv * per_head;
    const int rows_per_wg = max(1, 1024 / per_row), tiles = (a.budget + rows_per_wg - 1) / rows_per_wg;
    const int sl = (int)blockIdx.x / tiles, r0 = (int)blockIdx.x % tiles * rows_per_wg, b = a.b0 + sl;
    const int r1 = min(min(a.budget, a.n_rows[sl]), r0 + rows_per_wg);
    const size_t kld = (size_t)a.Hkv * a.dim;
    const int *from = a.pool.table + (size_t)b * a.pool.table_stride, *to = a.table_out + (size_t)b * a.pool.table_stride;
    for (int e = threadIdx.x; e < (r1 - r0) * per_row; e += 256) {
        const int j = r0 + e / per_row, c = e % per_row, h = c / per_head;
        const int src = pool_row(a.pool, from, a.kept[((size_t)b * a.Hkv + h) * a.budget + j]);
        const int dst = pool_row(a.pool, to, j);
        if (src < 0 || dst < 0) continue;
        const size_t s = (size_t)src * kld + (size_t)c * N, d = (size_t)dst * kld + (size_t)c * N;
        const vec x = *reinterpret_cast<const vec *>(a.pool.k + s), y = *reinterpret_cast<const vec *>(a.pool.v + s);
        *reinterpret_cast<vec *>(a.pool.k + d) = x;
        *reinterpret_cast<vec *>(a.pool.v + d) = y;
    }
}
extern "C" __global__ void __launch_bounds__(256) zt_evict_copy_4(PagedEvictArgs a) { evict_copy<4>(a); }
extern "C" __global__ void __launch_bounds__(256) zt_evict_copy_2(PagedEvictArgs a) { evict_copy<2>(a); }

// Rows within their own pages: a kept row only moves down, over rows that are gone or
// have moved already.  A thread owns N columns of K or V of one (sequence, kv head) for
// every row and no other wave touches its columns, so that all it takes is a wave's own order: of the 64 / L
// x U rows that a wave moves at a time every one is read before the first is written.
template <int N, int U>
DEVI void evict_move(const PagedEvictArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int per_head = a.dim / N;              // column pieces of a head's row
    const int L = 8, G = 64 / L;                 // lanes on a row, rows at a time
    const int parts = (per_head + L - 1) / L;
    int item = wave;
    const int part = item % parts;
    item /= parts;
    const bool is_v = item & 1;
    item >>= 1;
    const int h = item % a.Hkv, sl = item / a.Hkv;
    if (sl >= a.ns) return;  // wave-uniform
    const int b = a.b0 + sl;
    if (a.n_rows[sl] <= a.budget) return;
    const int *kept = a.kept + ((size_t)b * a.Hkv + h) * a.budget;
    const int *table = a.pool.table + (size_t)b * a.pool.table_stride;
    const size_t kld = (size_t)a.Hkv * a.dim;
    const int g = lane / L, c = part * L + lane % L;
    float *base = (is_v ? a.pool.v : a.pool.k) + (size_t)h * a.dim + (size_t)min(c, per_head - 1) * N;
    for (int j0 = 0; j0 < a.budget; j0 += G * U) {
        vec x[U];
        int dst[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + G * u + g;
            const int i = j < a.budget ? kept[j] : 0;
            dst[u] = -1;
            if (j < a.budget && i != j && c < per_head) {
                const int src = pool_row(a.pool, table, i);
                if (src >= 0) {
                    dst[u] = pool_row(a.pool, table, j);
                    x[u] = *reinterpret_cast<const vec *>(base + (size_t)src * kld);
                }
            }
        }
        wait_dma();  // every lane's reads are in registers before any lane writes
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (dst[u] >= 0) *reinterpret_cast<vec *>(base + (size_t)dst[u] * kld) = x[u];
    }
}
extern "C" __global__ void __launch_bounds__(256) zt_evict_move_4(PagedEvictArgs a) { evict_move<4, 8>(a); }
extern "C" __global__ void __launch_bounds__(256) zt_evict_move_2(PagedEvictArgs a) { evict_move<2, 8>(a); }
