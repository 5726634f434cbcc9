// Attention over a paged KV cache (gfx950): chunks of new tokens of a ragged batch of
// sequences, one token and more each, f32.
//
// For token t of a sequence (row R = n_rows - q_len + t of its cache) and query head h:
//     s_j = q_t . k_j / sqrt(d),  out = sum_{j <= R} softmax(s)_j v_j,  lse = log sum_j e^{s_j},
// rows k_j, v_j found through the sequence's page table.  The rows of one (sequence, kv
// head) are its tokens' query heads of that group, token-major, so a group's heads share
// every K and V row read, and a 16-row matrix tile is full from 16 / G tokens on.
//
// A page number outside the pool is never followed: a row that sees such a key comes
// out NaN.  A key that a row must not see gets the score -inf, and where a tile
// holds such a pair, V's values that are not finite are kept out of the products (0 x inf)
// and added to the rows that see them: nothing hidden reaches an output.  (A hidden K value of 2^40
// or more beside such a q moves a tile's products to f32 in the split-operand kernel, so that visible
// ones may be rounded otherwise.)
#include "attn_paged.h"

// ---- Accumulated weights ---------------------------------------------------------------
//
// Few rows in one chunk (more: paged_merge).  Sequences without new tokens copy their weights.
extern "C" __global__ void __launch_bounds__(256) zt_paged_weights(PagedWeightArgs a) {
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int n = sq.n_rows, kpad = (n + 15) & ~15, rows = sq.q_len * a.G;
    const int per_head = (n + 1023) / 1024;
    const int item = (int)blockIdx.x - sq.first;
    const int kvh = item / per_head, key = (item % per_head) * 1024 + 4 * (int)threadIdx.x;
    if (key >= n) return;
    const float *sp = a.scores + sq.at0 + (size_t)kvh * rows * kpad + key;
    const float *st = a.stat + 2 * ((size_t)sq.q0 * a.H + kvh * a.G);
    const f4 sum = weights_of_few(sp, kpad, rows, a.G, n - sq.q_len, key, [&](int r) {
        const int t = r / a.G;
        return *reinterpret_cast<const f2 *>(st + 2 * ((size_t)t * a.H + r - t * a.G));
    });
    const size_t at = ((size_t)sq.b * a.Hkv + kvh) * a.w_stride + key;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (key + e < n) a.w_out[at + e] = a.w_in[at + e] + sum[e];
}

// Sums of consecutive keys (N of them, some possibly past the last) over a part of the rows: to the part's
// place, or, where there is one part only, to the weights.
template <class V>
DEVI void put_part(const PagedWeightArgs &a, const PagedSeq &sq, int kvh, int nparts, int part, int key, V sum) {
    constexpr int N = sizeof(V) / sizeof(float);
    if (nparts == 1) {
        const size_t at = ((size_t)sq.b * a.Hkv + kvh) * a.w_stride + key;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float x;
            if constexpr (N == 1) x = sum; else x = sum[e];
            if (key + e < sq.n_rows) a.w_out[at + e] = a.w_in[at + e] + x;
        }
    } else if (key < sq.n_rows) {  // (a whole f4 fits: the parts' rows are padded to 16 keys)
        const int kpad = (sq.n_rows + 15) & ~15;
        *reinterpret_cast<V *>(a.parts + a.parts0[sq.i] + ((size_t)kvh * nparts + part) * kpad + key) = sum;
    }
}

// Many rows: from the tiles that the attention stored.  A workgroup takes 128 keys of one
// (sequence, kv head) and a part of the rows; a wave two neighbouring key tiles, 2 KB a row tile, four
// row tiles in flight: lane (l16, grp) adds row l16's weights of keys 4 grp .. 4 grp + 3 over the row
// tiles, and the 16 rows' lanes are added at the end.  Bound: HBM, the scores read once (a 2048-row
// prompt of 32 heads, 268 MB, about 45 us, 6 TB/s).
extern "C" __global__ void __launch_bounds__(256) zt_paged_wcols(PagedWeightArgs a) {
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int n = sq.n_rows, rows = sq.q_len * a.G, seen0 = n - sq.q_len, ktiles = (n + 15) >> 4;
    const int nparts = (rows + a.part_rows - 1) / a.part_rows, ntiles = (n + 127) / 128;
    int item = (int)blockIdx.x - sq.first;
    const int kvh = item % a.Hkv;
    item /= a.Hkv;
    const int part = nparts - 1 - item / ntiles, kt0 = item % ntiles * 128;
    if (max(0, kt0 - seen0) * a.G >= (part + 1) * a.part_rows) return;  // no row sees the keys; wsum skips it
    const int lane = lane_id(), l16 = lane & 15, grp = lane >> 4;
    const int k0 = kt0 + 32 * __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (k0 >= n) return;
    const int rt0 = max(part * a.part_rows, max(0, k0 - seen0) * a.G) >> 4;
    const int rt1 = (min(rows, (part + 1) * a.part_rows) + 15) >> 4;
    const bool two = k0 + 16 < n;
    const float *sp = a.scores + sq.at0 + 4 * lane + ((size_t)kvh * ((rows + 15) >> 4) * ktiles + (k0 >> 4)) * 256;
    const float *st = a.stat + 2 * ((size_t)sq.q0 * a.H + kvh * a.G);
    f4 sum[2] = {zero4(), zero4()};
    for (int rt = rt0; rt < rt1; rt += 4) {
        f4 s[4][2];
        f2 ml[4];
        int last[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = 16 * (rt + j) + l16, t = r / a.G;
            const bool in = r < rows && rt + j < rt1;
            last[j] = in ? seen0 + t : -1;
            ml[j] = f2{0.f, 0.f};
            if (in) ml[j] = *reinterpret_cast<const f2 *>(st + 2 * ((size_t)t * a.H + r - t * a.G));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[j][i] = zero4();
                // Tiles that none of their rows sees are not written.
                if (rt + j < rt1 && (i == 0 || two) && k0 + 16 * i <= seen0 + min(rows - 1, 16 * (rt + j) + 15) / a.G)
                    s[j][i] = __builtin_nontemporal_load(
                        reinterpret_cast<const f4 *>(sp + ((size_t)(rt + j) * ktiles + i) * 256));
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = k0 + 16 * i + 4 * grp;
            f4 four = zero4();
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    four[e] += key + e <= last[j] ? fast_exp2(s[j][i][e] - ml[j].x) * ml[j].y : 0.f;
            sum[i] += four;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 1; m < 16; m <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[i][e] += wave_xor(sum[i][e], m);
    if (l16 > 1 || (l16 == 1 && !two)) return;
    put_part(a, sq, kvh, nparts, part, k0 + 16 * l16 + 4 * grp, l16 ? sum[1] : sum[0]);
}

// Many rows whose scores are not kept: the scores again, on split operands.  A workgroup takes one (sequence, kv
// head, tile of 16 NK NW keys, part of the rows); a wave holds 16 NK keys (K's parts in registers), and Q
// passes through LDS in 32-row tiles, split once for all waves, two buffers, beside the rows'
// statistics.  S = Q K^T has a key per lane and four rows, so that the sum over rows
// stays in the lane until the end: in 32 bits over 64 tiles, those sums in 64 bits, so that
// its error does not grow with the rows (2^20 rows of weight 0.65 in 32 bits alone were off by 3.3e-4).
template <int DP, int NW, int NK, bool FULL>
DEVI void paged_wparts(const PagedWeightArgs &a) {
    constexpr int NKS = DP / 32, NTH = 64 * NW, TILE = split_bytes(DP, 32), KT = 16 * NK * NW;
    __shared__ __attribute__((aligned(16))) char smem[2 * TILE];
    __shared__ __attribute__((aligned(16))) float row_m[2][32], row_inv[2][32];
    __shared__ __attribute__((aligned(16))) int row_last[2][32];
    __shared__ int flags[2];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int n = sq.n_rows, q_len = sq.q_len, rows = q_len * a.G, seen0 = n - q_len;
    const int nparts = (rows + a.part_rows - 1) / a.part_rows;
    int item = (int)blockIdx.x - sq.first;
    const int kvh = item % a.Hkv;
    item /= a.Hkv;
    // Part by part, the last, which all keys of a prompt have rows in, first (neighbours of like length, as in
    // paged_many).
    const int ntiles = (n + KT - 1) / KT, part = nparts - 1 - item / ntiles, kt0 = item % ntiles * KT;
    // Rows of the part that see the tile's first key.
    const int r0 = max(part * a.part_rows, max(0, kt0 - seen0) * a.G) & ~31, r1 = min(rows, (part + 1) * a.part_rows);
    if (r0 >= r1) return;  // workgroup-uniform; zt_paged_wsum does not read it
    const int *table = a.pool.table + (size_t)sq.b * a.pool.table_stride;
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    const float *kb = a.pool.k + (size_t)kvh * a.dim;
    const bool vec4 = (a.dim & 3) == 0;
    if (tid < 2) flags[tid] = -1;

    const int k0 = kt0 + 16 * NK * w;  // the wave's first key
    Tri k[NKS][NK];
    float acc[NK], kmax = 0.f;
    double total[NK];
    const float *krow[NK];  // (null: a key without a page, whose scores are NaN)
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        acc[i] = 0.f;
        total[i] = 0.0;
        const int r = pool_row(a.pool, table, min(k0 + 16 * i + l16, n - 1));
        krow[i] = r < 0 ? nullptr : kb + (size_t)r * kld;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            float y[8];
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                float z[4];
                load_cols<4, FULL, false>(z, kb + (size_t)max(r, 0) * kld, 32 * ks + 8 * grp + h, a.dim, vec4);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[h + e] = r < 0 ? __builtin_nanf("") : z[e];
            }
            const float mx = max_abs(y);
            kmax = vmax(kmax, mx);
            if (any_big(mx)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = small_part(y[e]);
            }
            k[ks][i] = split8_as_is(y);
        }
    }
    const bool kbig = any_big(kmax);

    constexpr int CPR = DP / 8, CH = 32 * CPR, NP = (CH + NTH - 1) / NTH;
    constexpr bool EVEN = CH % NTH == 0;
    auto q_row = [&](int r) {  // of row r, or the part's last
        r = min(r, r1 - 1);
        const int t = r / a.G;
        return a.q + (size_t)(sq.q0 + t) * qld + (size_t)(kvh * a.G + r - t * a.G) * a.dim;
    };
    float px[NP][8], sm = 0.f, si = 0.f;
    int sl = 0;
    auto fetch = [&](int rt) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int e = tid + i * NTH;
            if (!EVEN && e >= CH) break;  // wave-uniform
            const float *p = q_row(rt + e / CPR);
#pragma unroll
            for (int h = 0; h < 8; h += 4) {
                float z[4];
                load_cols<4, FULL, false>(z, p, e % CPR * 8 + h, a.dim, vec4);
#pragma unroll
                for (int x = 0; x < 4; ++x) px[i][h + x] = z[x] * a.scale_log2e;
            }
        }
        if (tid < 32) {
            const int r = min(rt + tid, r1 - 1), t = r / a.G;
            const size_t row = (size_t)(sq.q0 + t) * a.H + kvh * a.G + r - t * a.G;
            const f2 ml = *reinterpret_cast<const f2 *>(a.stat + 2 * row);
            sm = ml.x;
            si = ml.y;
            sl = rt + tid < r1 ? seen0 + t : -1;  // a row past the part's last sees nothing
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int e = tid + i * NTH;
            if (!EVEN && e >= CH) break;
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = px[i][x];
            if (any_big(max_abs(y))) {
#pragma unroll
                for (int x = 0; x < 8; ++x) y[x] = small_part(y[x]);
                if (lane == 0) flags[buf & 1] = buf;
            }
            put_tri<DP>(smem + (buf & 1) * TILE, 32, e / CPR, e % CPR * 8, split8_as_is(y));
        }
        if (tid < 32) {
            row_m[buf & 1][tid] = sm;
            row_inv[buf & 1][tid] = si;
            row_last[buf & 1][tid] = sl;
        }
    };
    const int nsteps = (r1 - r0 + 31) >> 5;
    fetch(r0);
    __syncthreads();  // the flags
    put(0);
    if (nsteps > 1) fetch(r0 + 32);
    __syncthreads();
    for (int id = 0; id < nsteps; ++id) {
        const char *const Qs = smem + (id & 1) * TILE;
        const int rt = r0 + 32 * id;
        f4 s[2 * NK];  // s[j NK + i]: rows rt + 16 j + 4 grp + x, key k0 + 16 i + l16
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) s[i] = zero4();
        stream_parts<2 * NKS, 3>(
            [&](int i, int p) { return get_row<DP>(Qs, 32, 16 * (i / NKS), 32 * (i % NKS), l16, grp, p); },
            [&](int i, auto p, u4 x) {
                f4 t[NK];
#pragma unroll
                for (int j = 0; j < NK; ++j) t[j] = s[(i / NKS) * NK + j];
                mfma_parts<p>(t, x, [&](int j) -> const Tri & { return k[i % NKS][j]; });
#pragma unroll
                for (int j = 0; j < NK; ++j) s[(i / NKS) * NK + j] = t[j];
            });
        const bool qbig = __builtin_amdgcn_readfirstlane(flags[id & 1]) == id;
        if (kbig || qbig) {  // products with a big operand, from the full values; of both sides, all in f32
            if (kbig && qbig) {
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) s[i] = zero4();
            }
            const int ll = opaque(lane), lrow = ll & 15, lgrp = ll >> 4;
            const float *qrow[2] = {q_row(rt + lrow), q_row(rt + 16 + lrow)};
#pragma unroll 1
            for (int cc = 0; cc < 8 * NKS; ++cc) {
                const int col = 32 * (cc >> 3) + 8 * lgrp + (cc & 7);
                float kv[NK], qv[2];
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    kv[i] = !krow[i] ? __builtin_nanf("") : col < a.dim ? krow[i][col] : 0.f;
                    if (!qbig) kv[i] = big_part(kv[i]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qv[j] = col < a.dim ? qrow[j][col] * a.scale_log2e : 0.f;
                    if (!kbig) qv[j] = big_part(qv[j]);
                }
#pragma unroll
                for (int i = 0; i < 2 * NK; ++i) s[i] = mfma16(qv[i / NK], kv[i % NK], s[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int at = 16 * j + 4 * grp;
            const f4 m4 = *reinterpret_cast<const f4 *>(&row_m[id & 1][at]);
            const f4 i4 = *reinterpret_cast<const f4 *>(&row_inv[id & 1][at]);
            int last[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) last[x] = row_last[id & 1][at + x];
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int key = k0 + 16 * i + l16;
                float sum = 0.f;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float p = fast_exp2(s[j * NK + i][x] - m4[x]) * i4[x];
                    sum += key <= last[x] ? p : 0.f;
                }
                acc[i] += sum;
            }
        }
        if ((id & 63) == 63) {
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                total[i] += acc[i];
                acc[i] = 0.f;
            }
        }
        if (id + 1 < nsteps) {
            put(id + 1);
            if (id + 2 < nsteps) fetch(rt + 64);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const float sum = sum4grp((float)(total[i] + acc[i]));
        if (grp == 0) put_part(a, sq, kvh, nparts, part, k0 + 16 * i + l16, sum);
    }
}

// The parts of the rows, where there are several (2048 or so at most), added in order, in 64 bits.
template <int KT>
DEVI void paged_wsum(const PagedWeightArgs &a) {
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int n = sq.n_rows, q_len = sq.q_len, rows = q_len * a.G, kpad = (n + 15) & ~15;
    const int nparts = (rows + a.part_rows - 1) / a.part_rows;
    const int per_head = (n + 255) / 256;
    const int item = (int)blockIdx.x - sq.first;
    const int kvh = item / per_head, key = (item % per_head) * 256 + (int)threadIdx.x;
    if (key >= n) return;
    const int from = max(0, key / KT * KT - (n - q_len)) * a.G / a.part_rows;  // the first part that saw the tile
    const float *p = a.parts + a.parts0[sq.i] + (size_t)kvh * nparts * kpad + key;
    double sum = 0.0;
    for (int i = from; i < nparts; ++i) sum += p[(size_t)i * kpad];
    const size_t at = ((size_t)sq.b * a.Hkv + kvh) * a.w_stride + key;
    a.w_out[at] = (float)(a.w_in[at] + sum);
}

// (d = 256: one wave per SIMD, since two spill; 64 sequences of 2048 to 4096 rows of 16 over 4 heads 394 -> 290 us.)
#define ZT_PAGED_FEW(DP, NQ)                                                                        \
    extern "C" __global__ void __launch_bounds__(256, (DP) == 256 ? 1 : 2) zt_paged_few_d##DP##_n##NQ(PagedArgs a) {   \
        paged_few<DP, NQ, true>(a);                                                                 \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256, (DP) == 256 ? 1 : 2) zt_paged_few_d##DP##_n##NQ##_any(PagedArgs a) { \
        paged_few<DP, NQ, false>(a);                                                                \
    }
#define ZT_PAGED_MANY(DP, NW, NQ)                                                                   \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_paged_many_d##DP##_##NW##NQ(PagedArgs a) { \
        paged_many<DP, NW, NQ, true>(a);                                                            \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_paged_many_d##DP##_##NW##NQ##_any(PagedArgs a) { \
        paged_many<DP, NW, NQ, false>(a);                                                           \
    }
#define ZT_PAGED(DP)                                                                                \
    ZT_PAGED_FEW(DP, 1)                                                                             \
    extern "C" __global__ void __launch_bounds__(256) zt_paged_merge_d##DP(PagedArgs a) {     \
        paged_merge<DP, false>(a);                                                                  \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) zt_paged_merge_rows_d##DP(PagedArgs a) {       \
        paged_merge<DP, true>(a);                                                                   \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) zt_paged_merge_w_d##DP(PagedArgs a) {          \
        paged_merge<DP, false, true>(a);                                                            \
    }
ZT_PAGED(32)
ZT_PAGED(64)
ZT_PAGED(96)
ZT_PAGED(128)
ZT_PAGED(192)
ZT_PAGED(256)
ZT_PAGED_MANY(32, 4, 1) ZT_PAGED_MANY(32, 4, 2) ZT_PAGED_MANY(32, 8, 2)
ZT_PAGED_MANY(64, 4, 1) ZT_PAGED_MANY(64, 4, 2) ZT_PAGED_MANY(64, 8, 2)
ZT_PAGED_MANY(96, 4, 1) ZT_PAGED_MANY(96, 4, 2) ZT_PAGED_MANY(96, 8, 2)
ZT_PAGED_MANY(128, 4, 1) ZT_PAGED_MANY(128, 4, 2) ZT_PAGED_MANY(128, 8, 2)
ZT_PAGED_MANY(192, 4, 1) ZT_PAGED_MANY(192, 8, 1)
ZT_PAGED_MANY(256, 8, 1)
ZT_PAGED_FEW(32, 2) ZT_PAGED_FEW(64, 2) ZT_PAGED_FEW(96, 2) ZT_PAGED_FEW(128, 2)
#define ZT_PAGED_WPARTS(DP, NW, NK)                                                                 \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_paged_wparts_d##DP(PagedWeightArgs a) { \
        paged_wparts<DP, NW, NK, true>(a);                                                          \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_paged_wparts_d##DP##_any(PagedWeightArgs a) { \
        paged_wparts<DP, NW, NK, false>(a);                                                         \
    }
ZT_PAGED_WPARTS(32, 4, 2)
ZT_PAGED_WPARTS(64, 4, 2)
ZT_PAGED_WPARTS(96, 4, 2)
ZT_PAGED_WPARTS(128, 4, 2)
ZT_PAGED_WPARTS(192, 4, 1)
ZT_PAGED_WPARTS(256, 8, 1)
extern "C" __global__ void __launch_bounds__(256) zt_paged_wsum_128(PagedWeightArgs a) { paged_wsum<128>(a); }
extern "C" __global__ void __launch_bounds__(256) zt_paged_wsum_64(PagedWeightArgs a) { paged_wsum<64>(a); }
