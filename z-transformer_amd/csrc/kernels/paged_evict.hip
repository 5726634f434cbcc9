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

// Lane i of a row of 16 ends with the sum of the row's lanes 0 .. i (VALU only).
DEVI int row_scan(int v) {
    v += __builtin_amdgcn_mov_dpp(v, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8; 0 comes in
    v += __builtin_amdgcn_mov_dpp(v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x118, 0xf, 0xf, true);
    return v;
}
// From each wave's entry of red: the sum of those before wave w, and of all.
template <int NW>
DEVI int waves_before(const int *red, int w, int *all) {
    const int i = lane_id() & 15;
    const int v = row_scan(i < NW ? red[i] : 0);
    *all = __builtin_amdgcn_readlane(v, 15);
    return w ? __builtin_amdgcn_readlane(v, w - 1) : 0;
}
// The same, the wave's own number first put there.
template <int NW>
DEVI int block_before(int mine, int w, int *red, int *all) {
    __syncthreads();  // the last use's reads
    if (lane_id() == 0) red[w] = mine;
    __syncthreads();
    return waves_before<NW>(red, w, all);
}

// Lane i ends with the sum of the wave's lanes 0 .. i.
DEVI int wave_scan(int v) {
    v = row_scan(v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
    return v;
}

// Which rows stay: one workgroup of NW waves per (sequence, kv head).  With the candidates'
// weights as ordered numbers, T is the largest key that at least `need` of them reach, found by
// digits of 11, 11 and 10 bits: a histogram (LDS) of the digit among those that share the digits
// before it, summed from the top, says in which bin the need-th lies.  It ends early
// where a bin holds exactly as many as are wanted.  Those past T stay and, of those that equal
// it, the lowest rows that are still wanted.
//   KPT > 0, up to 64 NW KPT rows: a wave holds a run of 64 KPT rows in registers, so that w is read once, and
// two sums over the waves place every row.
//   KPT 0, any number: w is read again for every digit, and rows are placed 64 NW at a time, in order.
// w may be compacted in place: what a step overwrites has been read, since a row never moves up.
// Bound: latency, a few trips through LDS to a digit: 128 heads of up to 8192 rows 13 us (72 by single bits that read
// w again, 39 by two bits at a time, counted by ballots, from registers).
template <int NW, int KPT>
DEVI void evict_select(const PagedEvictArgs &a) {
    constexpr int NTH = 64 * NW, BINS = 2048, BPT = BINS / NTH;
    __shared__ __attribute__((aligned(16))) int hist[BINS];
    __shared__ int red[2][NW], found[3];
    const int tid = threadIdx.x, lane = lane_id(), wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sl = (int)blockIdx.x / a.Hkv, h = (int)blockIdx.x % a.Hkv, b = a.b0 + sl;
    const int n = a.n_rows[sl];
    const size_t head = (size_t)b * a.Hkv + h;
    const float *w = a.w_in + head * a.w_stride;
    float *wo = a.w_out + head * a.w_stride;
    int *kept = a.kept + head * a.budget;
    if (n <= a.budget) {  // all stay
        for (int i = tid; i < a.budget; i += NTH) kept[i] = i < n ? i : -1;
        if (wo != w)
            for (int i = tid; i < n; i += NTH) wo[i] = w[i];
        return;
    }
    const int lo = a.n_first, hi = n - a.n_last, need = a.budget - a.n_first - a.n_last;
    const int run0 = wv * 64 * KPT + lane;  // KPT > 0: the thread's rows are run0 + 64 k
    float x[KPT > 0 ? KPT : 1];
    unsigned key[KPT > 0 ? KPT : 1];
#pragma unroll
    for (int k = 0; k < KPT; ++k) {
        const int i = run0 + 64 * k;
        x[k] = i < n ? w[i] : 0.f;
        key[k] = weight_key(x[k]);
    }
    unsigned T = 0xffffffffu;  // that none reaches: a NaN's key is 0, +inf's less than this
    int equal = 0;             // rows wanted of those that equal T
    if (need > 0) {
        T = 0;
        equal = need;
        int left = 32;  // bits not looked at yet
        while (left > 0) {
            const int bits = left > 10 ? 11 : 10, shift = left - bits;
#pragma unroll
            for (int j = 0; j < BPT; ++j) hist[j * NTH + tid] = 0;
            __syncthreads();
            auto put = [&](unsigned ki) {  // a candidate; those that share the digits so far count
                if (left == 32 || ki >> left == T >> left) atomicAdd(&hist[ki >> shift & ((1 << bits) - 1)], 1);
            };
            if constexpr (KPT > 0) {
#pragma unroll
                for (int k = 0; k < KPT; ++k) {
                    const int i = run0 + 64 * k;
                    if (i >= lo && i < hi) put(key[k]);
                }
            } else {
                for (int i = lo + tid; i < hi; i += NTH) put(weight_key(w[i]));
            }
            __syncthreads();
            // From the top: thread t has bins BINS - 1 - BPT t and below.
            int c[BPT], sum = 0;
#pragma unroll
            for (int j = 0; j < BPT; ++j) {
                c[j] = hist[BINS - 1 - (BPT * tid + j)];
                sum += c[j];
            }
            const int upto = wave_scan(sum);
            if (lane == 63) red[0][wv] = upto;
            __syncthreads();
            int all;
            int above = waves_before<NW>(red[0], wv, &all) + upto - sum;
#pragma unroll
            for (int j = 0; j < BPT; ++j) {
                if (above < equal && above + c[j] >= equal) {  // one thread's one bin
                    found[0] = BINS - 1 - (BPT * tid + j);
                    found[1] = above;
                    found[2] = c[j];
                }
                above += c[j];
            }
            __syncthreads();
            T |= (unsigned)found[0] << shift;
            equal -= found[1];
            left = shift;
            if (found[2] == equal) {  // all that reach T stay, whatever the bits behind it
                if (T == 0) break;    // (every candidate, NaN among them: those equal to 0 by row are all)
                --T;
                equal = 0;
                break;
            }
        }
    }
    const unsigned long long below = (1ull << lane) - 1;
    if constexpr (KPT > 0) {
        int eq = 0, all = 0;
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const int i = run0 + 64 * k;
            eq += __popcll(__builtin_amdgcn_ballot_w64(i >= lo && i < hi && key[k] == T));
        }
        int eq_at = block_before<NW>(eq, wv, red[0], &all);
        unsigned long long stay[KPT];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const int i = run0 + 64 * k;
            const bool cand = i >= lo && i < hi;
            const unsigned long long e = __builtin_amdgcn_ballot_w64(cand && key[k] == T);
            stay[k] = __builtin_amdgcn_ballot_w64(
                i < n && (!cand || key[k] > T || (key[k] == T && eq_at + __popcll(e & below) < equal)));
            eq_at += __popcll(e);
            mine += __popcll(stay[k]);
        }
        int at = block_before<NW>(mine, wv, red[1], &all);
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            if (stay[k] >> lane & 1) {
                const int to = at + __popcll(stay[k] & below);
                kept[to] = run0 + 64 * k;
                wo[to] = x[k];
            }
            at += __popcll(stay[k]);
        }
    } else {
        int n_kept = 0, n_equal = 0;
        for (int i0 = 0; i0 < n; i0 += NTH) {
            const int i = i0 + tid;
            const float wi = i < n ? w[i] : 0.f;
            const bool cand = i >= lo && i < hi;
            const unsigned ki = weight_key(wi);
            const unsigned long long eq = __builtin_amdgcn_ballot_w64(cand && ki == T);
            int all_eq = 0;
            const int eq_before = block_before<NW>(__popcll(eq), wv, red[0], &all_eq) + n_equal;
            const bool keep = i < n && (!cand || ki > T || (ki == T && eq_before + __popcll(eq & below) < equal));
            const unsigned long long st = __builtin_amdgcn_ballot_w64(keep);
            int all = 0;
            const int at = block_before<NW>(__popcll(st), wv, red[1], &all) + n_kept + __popcll(st & below);
            if (keep) {
                kept[at] = i;
                wo[at] = wi;
            }
            n_kept += all;
            n_equal += all_eq;
        }
    }
}

#define ZT_EVICT_SELECT(NAME, NW, KPT)                                                              \
    extern "C" __global__ void __launch_bounds__(64 * NW) zt_evict_select_##NAME(PagedEvictArgs a) { \
        evict_select<NW, KPT>(a);                                                                   \
    }
ZT_EVICT_SELECT(1024, 4, 4)
ZT_EVICT_SELECT(4096, 8, 8)
ZT_EVICT_SELECT(16384, 16, 16)
ZT_EVICT_SELECT(any, 16, 0)

// Rows to other pages: a thread takes 4 N bytes of K and V at a time.  Bound: HBM, a copy (16 sequences of up to
// 8192 rows to 4096, 8 kv heads at d = 128, 220 us: 4.7 TB/s, as a copy of 4 GiB).
template <int N>
DEVI void evict_copy(const PagedEvictArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    const int per_head = a.dim / N, per_row = a.Hkv * per_head;
    const int rows_per_wg = max(1, 1024 / per_row);
    const int sl = (int)blockIdx.x / a.tiles, r0 = (int)blockIdx.x % a.tiles * rows_per_wg, b = a.b0 + sl;
    const int r1 = min(min(a.budget, a.n_rows[sl]), r0 + rows_per_wg);
    const size_t kld = (size_t)a.Hkv * a.dim;
    const size_t entry = (size_t)b * a.pool.table_stride;
    const int *from = a.pool.table + entry, *to = a.table_out + entry;
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
// have moved already.  A workgroup takes K or V of one (sequence, kv head) and walks the rows upwards, a tile of
// 4 x 1024 16-byte (8-byte) pieces at a time: all of a tile's rows are in registers, in every
// wave, before one is written, and what a later tile reads lies past all that earlier ones write.
// Bound: HBM for many sequences, the tiles' trips to memory one after the other for few: 8 kv heads at d = 128,
// 8192 rows cut to 4096, 16 sequences 234 us (4.6 TB/s), one 70; with a wave to 64 rows of 128 bytes at a time
// instead 555 and 311, with 8 x 512 pieces 239 and 80.
template <int N>
DEVI void evict_move(const PagedEvictArgs &a) {
    typedef float vec __attribute__((ext_vector_type(N)));
    constexpr int U = 4;
    const int is_v = (int)blockIdx.x & 1, h = ((int)blockIdx.x >> 1) % a.Hkv, sl = ((int)blockIdx.x >> 1) / a.Hkv;
    const int b = a.b0 + sl;
    if (a.n_rows[sl] <= a.budget) return;  // workgroup-uniform
    const int *kept = a.kept + ((size_t)b * a.Hkv + h) * a.budget;
    const int *table = a.pool.table + (size_t)b * a.pool.table_stride;
    const size_t kld = (size_t)a.Hkv * a.dim;
    const int per_head = a.dim / N, rows = 1024 / per_head;  // rows of a pass
    const int r = (int)threadIdx.x / per_head, c = (int)threadIdx.x % per_head;
    float *base = (is_v ? a.pool.v : a.pool.k) + (size_t)h * a.dim + (size_t)c * N;
    int src[U], dst[U];
    auto places = [&](int j0) {  // of the thread's rows of the tile at j0; -1: nothing to move
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + rows * u + r, jc = min(j, a.budget - 1), i = kept[jc];
            const bool moves = r < rows && j < a.budget && i != j;
            const int from = pool_row(a.pool, table, i), to = pool_row(a.pool, table, jc);
            src[u] = moves ? from : -1;
            dst[u] = to;
        }
    };
    places(0);
    for (int j0 = 0; j0 < a.budget; j0 += rows * U) {
        vec x[U];
        int to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            to[u] = src[u] >= 0 ? dst[u] : -1;
            if (to[u] >= 0) x[u] = *reinterpret_cast<const vec *>(base + (size_t)src[u] * kld);
        }
        places(j0 + rows * U);  // the next tile's
        wait_dma();
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (to[u] >= 0) *reinterpret_cast<vec *>(base + (size_t)to[u] * kld) = x[u];
    }
}
extern "C" __global__ void __launch_bounds__(1024) zt_evict_move_4(PagedEvictArgs a) { evict_move<4>(a); }
extern "C" __global__ void __launch_bounds__(1024) zt_evict_move_2(PagedEvictArgs a) { evict_move<2>(a); }
