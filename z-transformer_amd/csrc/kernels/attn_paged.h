// Attention over a paged KV cache (gfx950), f32: the kernels' bodies, for chunks of new tokens (attn_paged.hip) and, with
// TREE, for trees of drafted ones (attn_tree.hip).
#pragma once
#include "common.h"
#include "args.h"
#include "paged.h"
#include "split.h"

// N consecutive floats (2 or 4) of a row at column c; FULL: the row has DP aligned
// columns; else columns past dim are 0 and rows may be 8-byte aligned only.  ONCE: read by one
// workgroup only, and kept out of the caches (a prompt, whose workgroups share its K and V rows, 667 us so, 653 not).
template <int N, bool FULL, bool ONCE>
DEVI void load_cols(float *dst, const float *row, int c, int dim, bool vec4) {
    if constexpr (N == 4) {
        f4 x = zero4();
        if (FULL || (vec4 && c < dim)) {
            const f4 *p = reinterpret_cast<const f4 *>(row + c);
            x = ONCE ? __builtin_nontemporal_load(p) : *p;
        } else if (!vec4) {
            if (c < dim) {
                const f2 y = *reinterpret_cast<const f2 *>(row + c);
                x.x = y.x; x.y = y.y;
            }
            if (c + 2 < dim) {
                const f2 y = *reinterpret_cast<const f2 *>(row + c + 2);
                x.z = y.x; x.w = y.y;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) dst[e] = x[e];
    } else {
        f2 x = f2{0.f, 0.f};
        if (FULL || c < dim) {
            const f2 *p = reinterpret_cast<const f2 *>(row + c);
            x = ONCE ? __builtin_nontemporal_load(p) : *p;
        }
        dst[0] = x.x; dst[1] = x.y;
    }
}

// ---- Trees of new tokens ---------------------------------------------------------------
//
// Token t's mask is 32-bit words, bit j of word j / 32 set where it sees new token j; no token sees a later
// one.  A token whose mask leaves nothing, in a cache that holds nothing else, comes out 0, its log-sum-exp -inf.

// Which of 32 keys the token (packed number `token`) sees by its mask, bit i: key k0 + i, the new tokens' keys
// beginning at seen0; k0 > seen0 - 32.  Bits past the mask's last word are 0.
DEVI unsigned tree_window(const PagedArgs &a, int token, int k0, int seen0) {
    const unsigned *m = a.mask + (size_t)token * a.mask_ld;
    const int off = k0 - seen0;
    if (off < 0) return m[0] << -off | ((1u << -off) - 1);  // (the keys before the new tokens' are seen by all)
    const int i = off >> 5;
    const unsigned lo = i < a.mask_ld ? m[i] : 0, hi = i + 1 < a.mask_ld ? m[i + 1] : 0;
    return __builtin_amdgcn_alignbit(hi, lo, off & 31);
}

// Whether new token t (packed number `token`) sees no key at all.
DEVI bool tree_sees_none(const PagedArgs &a, int token, int t, int seen0) {
    if (seen0 > 0) return false;
    const unsigned *m = a.mask + (size_t)token * a.mask_ld;
    unsigned any = 0;
    for (int i = 0; i < t >> 5; ++i) any |= m[i];
    return (any | (m[t >> 5] & ((2u << (t & 31)) - 1))) == 0;
}

// A row's statistics: log-sum-exp in natural units, base and inverse sum for its weights.
template <bool TREE>
DEVI void put_stats(const PagedArgs &a, size_t row, float m, float l) {
    if (a.lse) a.lse[row] = (m + log2f(l)) * 0.69314718055994531f;
    if (!TREE && a.stat) *reinterpret_cast<f2 *>(a.stat + 2 * row) = f2{m, 1.f / l};
}

// ---- Few rows: K and V stream through registers -----------------------------------
//
// A workgroup takes one (sequence, kv head, chunk of keys) and all of its rows, at most 16 NQ; its
// four waves take the chunk's 16-key tiles in turn.  Bound: HBM, each K and V row read once per kv
// head: a token of each of 64 sequences of 4096 to 8192 rows, 32 over 8 heads at d = 128, 505 us, 6.4 TB/s
// (a streaming read reaches 7.1), the matrix cores 39 % busy, with 1 row or 16.
//   * S^T = K Q^T on v_mfma_f32_16x16x4_f32 with the contraction dealt so that k-step
//     (j, e) of lane group grp is column 16 j + 4 grp + e: the A operand is then what
//     lane (l16, grp) loads of key l16 with 16-byte loads, straight from memory.
//   * O^T += V^T P^T in the row-owner layout (common.h): its A operand is what lane
//     (l16, grp) loads of keys 4 grp .. 4 grp + 3, 16 lanes on one row's consecutive chunks.
//   So no byte of K or V passes through LDS, and a row is read in whole 64- and 256-byte pieces.
//   * K of the next tile is loaded when this tile's scores are done, V after its
//     products: one buffer of each, always in flight during the other's half.
template <int DP, int NQ, bool FULL, bool TREE = false>
DEVI void paged_few(const PagedArgs &a) {
    constexpr int NT = DP / 16, C = ro_chunk<NT>(), NV = NT / C, NW = 4, LW = DP + 4;
    __shared__ float Wacc[NW][16][LW];
    __shared__ float Wm[NW][16], Wl[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int nch = sq.nch, q_len = sq.q_len, rows = q_len * a.G;  // at most 16 NQ rows
    const int item = (int)blockIdx.x - sq.first, c = item % nch, kvh = item / nch;
    const int seen0 = sq.n_rows - q_len;  // the cache row of token 0, the last it sees
    const int key0 = c * sq.chunk, key1 = min(sq.n_rows, key0 + sq.chunk);
    const int *table = a.pool.table + (size_t)sq.b * a.pool.table_stride;
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    const bool vec4 = (a.dim & 3) == 0;
    const float *kb = a.pool.k + (size_t)kvh * a.dim, *vb = a.pool.v + (size_t)kvh * a.dim;

    // Q: k-step (j, e) is column 16 j + 4 grp + e.  Rows past the last take its values; nothing of them is stored.
    float q[NQ][NT][4];
    int last[NQ];  // the last key that the lane's row sees
    unsigned tree[NQ];  // and which of the new tokens' keys (32 at most), if not all up to it
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = min(16 * n + l16, rows - 1), t = r / a.G;
        last[n] = seen0 + t;
        if constexpr (TREE) tree[n] = a.mask[(size_t)(sq.q0 + t) * a.mask_ld];
        const float *row = a.q + (size_t)(sq.q0 + t) * qld + (size_t)(kvh * a.G + r - t * a.G) * a.dim;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            load_cols<4, FULL, true>(q[n][j], row, 16 * j + 4 * grp, a.dim, vec4);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[n][j][e] *= a.scale_log2e;
        }
    }
    f4 o[NQ][NT];
    float m[NQ], lsum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int i = 0; i < NT; ++i) o[n][i] = zero4();
        m[n] = -INFINITY;
        lsum[n] = 0.f;
    }

    const int ntiles = (key1 - key0 + 15) >> 4;
    // Pool row of the lane's key (l16) of a tile; keys past the chunk's last stand on that one.
    auto row_of = [&](int t) { return pool_row(a.pool, table, min(key0 + 16 * t + l16, key1 - 1)); };
    float kx[NT][4], vx[4][NV][C];
    int vrow[4];
    auto load_k = [&](int row) {
        const float *p = kb + (size_t)max(row, 0) * kld;
#pragma unroll
        for (int j = 0; j < NT; ++j) load_cols<4, FULL, true>(kx[j], p, 16 * j + 4 * grp, a.dim, vec4);
    };
    auto load_v = [&](int row) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            vrow[r] = __shfl(row, 4 * grp + r, 64);
            const float *p = vb + (size_t)max(vrow[r], 0) * kld;
#pragma unroll
            for (int i = 0; i < NV; ++i) load_cols<C, FULL, true>(vx[r][i], p, 16 * C * i + C * l16, a.dim, vec4);
        }
    };
    auto in_tree = [&](int n, int key) { return key < seen0 || (tree[n] >> ((key - seen0) & 31) & 1); };
    int next = 0;
    if (w < ntiles) {
        const int row = row_of(w);
        load_k(row);
        load_v(row);
        next = row_of(min(w + NW, ntiles - 1));
    }
    for (int t = w; t < ntiles; t += NW) {
        const int k0 = key0 + 16 * t;
        const bool more = t + NW < ntiles;
        f4 s[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            f4 s0 = zero4(), s1 = zero4();  // two chains: one alone would wait for itself
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (j & 1) s1 = mfma16(kx[j][e], q[n][j][e], s1);
                    else s0 = mfma16(kx[j][e], q[n][j][e], s0);
                }
            s[n] = s0 + s1;
        }
        if (more) load_k(next);
        // Keys 4 grp + r of the tile are this lane's; hidden ones and those without a page.
        const bool edge = (TREE ? k0 + 15 >= seen0 : k0 + 15 > seen0) || k0 + 16 > key1;  // wave-uniform
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (vrow[r] < 0) s[n][r] = __builtin_nanf("");
                const int key = k0 + 4 * grp + r;
                if (edge && (key > last[n] || key >= key1)) s[n][r] = -INFINITY;
                if constexpr (TREE) {
                    if (edge && !in_tree(n, key)) s[n][r] = -INFINITY;
                }
            }
        if (!TREE && a.scores) {
            const int kpad = (sq.n_rows + 15) & ~15;
            float *sp = a.scores + a.score0[sq.i] + (size_t)kvh * rows * kpad + k0 + 4 * grp;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int r = 16 * n + l16;
                if (r < rows) *reinterpret_cast<f4 *>(sp + (size_t)r * kpad) = s[n];
            }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float y[4] = {s[n][0], s[n][1], s[n][2], s[n][3]};
            const float mt = max4grp(vmax_n(y));
            // The base is raised only when a score passes it by 2^8: weights stay under that.
            if (mt > m[n] + 8.f) {
                const float mnew = vmax(m[n], mt), corr = fast_exp2(m[n] - mnew);
                m[n] = mnew;
                lsum[n] *= corr;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[n][i] *= corr;
            }
            const float mb = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = fast_exp2(s[n][r] - mb);
            lsum[n] += (s[n][0] + s[n][1]) + (s[n][2] + s[n][3]);
        }
        // Where a pair is hidden, V's values that are not finite leave the products (their weight may be 0 for
        // being hidden) and are added one by one to the rows that see them.
        bool odd_v = false;
        if (edge) {
            bool odd = false;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < C; ++e) odd |= !(__builtin_fabsf(vx[r][i][e]) < INFINITY);
            odd_v = __builtin_amdgcn_ballot_w64(odd) != 0;
            if (odd_v) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int e = 0; e < C; ++e)
                            vx[r][i][e] = __builtin_fabsf(vx[r][i][e]) < INFINITY ? vx[r][i][e] : 0.f;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int n = 0; n < NQ; ++n) o[n][i] = mfma16(vx[r][i / C][i % C], s[n][r], o[n][i]);
        if (odd_v) {
            // The lane's columns of the key's V row, the weight from the lane group that holds it.
            const int ll = opaque(lane), lcol = ll & 15, lgrp = ll >> 4;
#pragma unroll 1
            for (int key = 0; key < 16; ++key) {
                const int vr = key & 2 ? (key & 1 ? vrow[3] : vrow[2]) : (key & 1 ? vrow[1] : vrow[0]);
                const int row = __shfl(vr, 16 * (key >> 2), 64);
                const float *p = vb + (size_t)max(row, 0) * kld;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float sr = key & 2 ? (key & 1 ? s[n][3] : s[n][2]) : (key & 1 ? s[n][1] : s[n][0]);
                    const float pk = __shfl(sr, 16 * (key >> 2) + lcol, 64);
                    bool sees = k0 + key <= last[n] && k0 + key < key1;
                    if constexpr (TREE) sees = sees && in_tree(n, k0 + key);
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int col = i / C * 16 * C + C * (4 * lgrp + r) + i % C;
                            if (!sees || (!FULL && col >= a.dim)) continue;
                            const float x = p[col];
                            if (!(__builtin_fabsf(x) < INFINITY)) o[n][i][r] += pk * x;
                        }
                }
            }
        }
        if (more) {
            load_v(next);
            next = row_of(min(t + 2 * NW, ntiles - 1));
        }
    }

    // The four waves' parts, rescaled to their largest base, added in wave order.
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float l = sum4grp(lsum[n]);
        if (n) __syncthreads();
        if (grp == 0) { Wm[w][l16] = m[n]; Wl[w][l16] = l; }
#pragma unroll
        for (int r = 0; r < 4; ++r) store_run<NT>(Wacc[w][l16], 4 * grp + r, DP, true, o[n], r, 1.f);
        __syncthreads();
        for (int e = tid; e < 16 * (DP / 4); e += 64 * NW) {
            const int i = e / (DP / 4), col = 4 * (e % (DP / 4)), r = 16 * n + i;
            if (r >= rows || col >= a.dim) continue;
            float M = Wm[0][i];
#pragma unroll
            for (int x = 1; x < NW; ++x) M = fmaxf(M, Wm[x][i]);
            float L = 0.f;
            f4 A = zero4();
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = Wm[x][i] == -INFINITY ? 0.f : fast_exp2(Wm[x][i] - M);
                L += Wl[x][i] * f;
                A += *reinterpret_cast<const f4 *>(&Wacc[x][i][col]) * f;
            }
            const int t = r / a.G, h = kvh * a.G + r - t * a.G;
            const size_t row = (size_t)(sq.q0 + t);
            if (nch == 1) {
                if (col == 0) {
                    put_stats<TREE>(a, row * a.H + h, M, L);
                }
                f4 y = A * (1.f / L);
                if (TREE && L == 0.f && tree_sees_none(a, (int)row, t, seen0)) y = zero4();
                store4(a.out + row * qld + (size_t)h * a.dim, col, a.dim, vec4, y);
            } else {
                const size_t slot = (size_t)sq.at0 + ((size_t)kvh * rows + r) * nch + c;
                *reinterpret_cast<f4 *>(a.part_acc + slot * a.part_ld + col) = A;
                if (col == 0) { a.part_ml[2 * slot] = M; a.part_ml[2 * slot + 1] = L; }
            }
        }
    }
}

// ---- Many rows: split operands -------------------------------------------------------
//
// The products on the bf16 matrix cores from three exact parts per operand (split.h).  A
// workgroup takes one (sequence, kv head, chunk of keys, tile of 16 NQ NW rows); a wave holds 16 NQ of the
// rows (Q's parts, O and the softmax state in registers), and the 32-key tiles of K and V pass through LDS,
// split once for all waves: two buffers of each, and the second half of the waves runs half a step behind the
// first, so that one half's softmax and splitting run beside the other's products.
//   A step is phase A (S^T = K Q^T, softmax; the next K tile into LDS) and phase B (O^T += V^T P^T; the
//   next V tile); tiles are loaded a whole step before they are written to LDS where registers allow (DEEP),
//   else in that phase.
//   * The pool rows that a thread stages are looked up in the page table one tile ahead of its loads.
//   * The rows of V hold a value that is big (split.h), or that is not finite where a pair of the tile is
//     hidden, as 0 in the split, and it is added from the full row to the rows that see it.
//   * A key whose page is none of the pool's is staged as NaN: the scores it meets are NaN.
// Bound: as the contiguous forward, the vector instructions beside the MFMAs, two to each, at two waves per SIMD:
// a prompt of 4096 rows, 32 over 8 heads at d = 128, 645 us, 213 TFLOP/s, the matrix cores 57 % busy.
template <int DP, int NW, int NQ>
struct PagedMany {
    static constexpr int NT = DP / 16, NKS = DP / 32, NTH = 64 * NW;
    static constexpr int TILE = split_bytes(DP, 32);
    static constexpr bool ALT = NW == 8 && 4 * TILE + 16 <= 160 * 1024;
    static constexpr bool DEEP = NQ == 1 || DP <= 64;
    static constexpr int FLAGS = (ALT ? 4 : 2) * TILE;
    static constexpr int BYTES = FLAGS + 16;
};

template <int DP, int NW, int NQ, bool FULL, bool TREE = false>
DEVI void paged_many(const PagedArgs &a) {
    using P = PagedMany<DP, NW, NQ>;
    constexpr int NT = P::NT, NKS = P::NKS, NTH = P::NTH;
    constexpr bool ALT = P::ALT, DEEP = P::DEEP;
    __shared__ __attribute__((aligned(16))) char smem[P::BYTES];
    // The K (V) tile of step id, and the flag that holds id if V's tile has values to add.
    auto ktile = [&](int id) { return smem + (ALT ? (id & 1) * 2 * P::TILE : 0); };
    auto vtile = [&](int id) { return ktile(id) + P::TILE; };
    int *const flags = reinterpret_cast<int *>(smem + P::FLAGS);
    auto kflag = [&](int id) { return flags + (ALT ? (id & 1) * 2 : 0); };
    auto vflag = [&](int id) { return kflag(id) + 1; };

    const int tid = opaque((int)threadIdx.x), lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int nch = sq.nch, q_len = sq.q_len, rows = q_len * a.G;
    int item = (int)blockIdx.x - sq.first;
    const int kvh = item % a.Hkv;
    item /= a.Hkv;
    // Chunk by chunk, in each the last row tile, with most keys, first: neighbours are of like length (workgroups
    // go to the XCDs and their shader engines in turn, so that a pattern of long and short ones would
    // pile up the long ones: a 2048-row prompt cut in two took 327 us with a tile's chunks side by side).
    constexpr int RT = 16 * NQ * NW;  // rows of a workgroup
    const int ntiles = (rows + RT - 1) / RT, c = item / ntiles;
    const int wg_row0 = (ntiles - 1 - item % ntiles) * RT, row0 = wg_row0 + 16 * NQ * w;
    const int seen0 = sq.n_rows - q_len;
    const int kend_wg = seen0 + (min(rows, wg_row0 + RT) - 1) / a.G + 1;
    const int kend_w = row0 < rows ? seen0 + (min(rows, row0 + 16 * NQ) - 1) / a.G + 1 : 0;
    const int key0 = c * sq.chunk, key1 = min(kend_wg, key0 + sq.chunk);
    if (key0 >= kend_wg) return;  // workgroup-uniform
    const int edge0 = TREE ? seen0 - 1 : seen0 + wg_row0 / a.G;  // the workgroup's rows see all keys up to this one
    const int *table = a.pool.table + (size_t)sq.b * a.pool.table_stride;
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    const float *kb = a.pool.k + (size_t)kvh * a.dim, *vb = a.pool.v + (size_t)kvh * a.dim;
    const bool vec4 = (a.dim & 3) == 0;
    if (tid < 4) flags[tid] = -1;

    // Staging: thread tid takes the 8-column chunks e = tid + n NTH of a 32-key tile.
    constexpr int CPR = DP / 8, CH = 32 * CPR, NP = (CH + NTH - 1) / NTH;
    constexpr bool EVEN = CH % NTH == 0;
    auto rows_of = [&](int (&r)[NP], int id) {  // pool rows of the chunks of step id; past the last key, that one's
#pragma unroll
        for (int n = 0; n < NP; ++n)
            r[n] = pool_row(a.pool, table, min(key0 + 32 * id + (tid + n * NTH) / CPR % 32, key1 - 1));
    };
    auto fetch = [&](float (&x)[NP][8], const float *base, const int (&r)[NP]) {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int e = tid + n * NTH;
            if (!EVEN && e >= CH) break;  // wave-uniform: CH is a multiple of 64
            const float *p = base + (size_t)max(r[n], 0) * kld;
            float y[4];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                load_cols<4, FULL, false>(y, p, e % CPR * 8 + i, a.dim, vec4);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[n][i + k] = y[k];
            }
        }
    };
    auto put = [&](const float (&x)[NP][8], char *t, int *flag, int id, bool odd_too, auto split) {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int e = tid + n * NTH;
            if (!EVEN && e >= CH) break;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[n][i];
            bool take = any_big(max_abs(y));
            if (odd_too) {
                bool nan = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) nan |= y[i] != y[i];
                take |= __builtin_amdgcn_ballot_w64(nan) != 0;
            }
            if (take) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = odd_too && y[i] != y[i] ? 0.f : small_part(y[i]);
                if (lane == 0) *flag = id;
            }
            put_tri<DP>(t, 32, e / CPR, e % CPR * 8, split(y));
        }
    };

    // Q: the B operand of the score product, lane l16 = row, k slot = column.  Rows past the last take its values.
    Tri q[NKS][NQ];
    int last[NQ];
    float qmax = 0.f;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = min(row0 + 16 * n + l16, rows - 1), t = r / a.G;
        last[n] = seen0 + t;
        const float *row = a.q + (size_t)(sq.q0 + t) * qld + (size_t)(kvh * a.G + r - t * a.G) * a.dim;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                float z[4];
                load_cols<4, FULL, false>(z, row, 32 * ks + 8 * grp + i, a.dim, vec4);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[i + k] = z[k] * a.scale_log2e;
            }
            const float mx = max_abs(y);
            qmax = vmax(qmax, mx);
            if (any_big(mx)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = small_part(y[i]);
            }
            q[ks][n] = split8_as_is(y);
        }
    }
    const bool qbig = any_big(qmax);
    f4 o[NT][NQ];
    float m[NQ], lsum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][n] = zero4();
        m[n] = -INFINITY;
        lsum[n] = 0.f;
    }

    f4 s[2 * NQ];  // s[j NQ + n]: keys k0 + 16 j + 4 grp + r of row block n
    auto windows = [&](unsigned (&x)[NQ], int k0) {  // tree_window of the lane's rows
#pragma unroll
        for (int n = 0; n < NQ; ++n) x[n] = k0 + 31 >= seen0 ? tree_window(a, sq.q0 + last[n] - seen0, k0, seen0) : ~0u;
    };
    unsigned tree[NQ];  // of the step at hand
    auto softmax = [&](const int k0) {
        if (TREE ? k0 + 31 >= seen0 || k0 + 32 > key1 : k0 + 31 > seen0 + row0 / a.G || k0 + 32 > key1) {  // wave-uniform
#pragma unroll
            for (int i = 0; i < 2 * NQ; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = 16 * (i / NQ) + 4 * grp + r, key = k0 + at;
                    if (key > last[i % NQ] || key >= key1 || (TREE && !(tree[i % NQ] >> at & 1))) s[i][r] = -INFINITY;
                }
        }
        if (!TREE && a.scores) {  // kept for the weights: 16 x 16 tiles as the lanes hold them, 1 KB a store
            const int ktiles = (sq.n_rows + 15) >> 4;
            float *sp = a.scores + a.score0[sq.i] + 4 * lane +
                        (((size_t)kvh * ((rows + 15) >> 4) + (row0 >> 4)) * ktiles + (k0 >> 4)) * 256;
#pragma unroll
            for (int i = 0; i < 2 * NQ; ++i)
                if (row0 + 16 * (i % NQ) < rows && k0 + 16 * (i / NQ) < key1) {  // wave-uniform
                    float *p = sp + ((size_t)(i % NQ) * ktiles + i / NQ) * 256;
                    __builtin_nontemporal_store(s[i], reinterpret_cast<f4 *>(p));
                }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = s[(i / 4) * NQ + n][i % 4];
            const float mt = max4grp(vmax_n(y));
            if (mt > m[n] + 8.f) {  // the base is raised only when a score passes it by 2^8
                const float mnew = vmax(m[n], mt), corr = fast_exp2(m[n] - mnew);
                m[n] = mnew;
                lsum[n] *= corr;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[i][n] *= corr;
            }
            const float mb = m[n] == -INFINITY ? 0.f : m[n];  // nothing seen yet
            float ps = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = fast_exp2(y[i] - mb);
                s[(i / 4) * NQ + n][i % 4] = y[i];
                ps = i == 0 ? y[0] : ps + y[i];
            }
            lsum[n] += ps;
        }
    };

    const int nsteps = (key1 - key0 + 31) >> 5;
    float px[NP][8], py[DEEP ? NP : 1][8];
    int rk[NP], rv[NP], rn[NP];  // pool rows of the next K fetch, of the next V fetch, and of the tile after
    const auto as_is = [](const float (&y)[8]) { return split8_as_is(y); };
    const auto scaled = [](const float (&y)[8]) { return split8(y); };
    auto copy_rows = [](int (&to)[NP], const int (&from)[NP]) {
#pragma unroll
        for (int n = 0; n < NP; ++n) to[n] = from[n];
    };
    bool none[NP];  // of the K tile in px: its page is none of the pool's
    auto fetch_k = [&](int id) {  // then the rows of the tile after it
        copy_rows(rk, rn);
        fetch(px, kb, rk);
#pragma unroll
        for (int n = 0; n < NP; ++n) none[n] = rk[n] < 0;
        rows_of(rn, min(id + 1, nsteps - 1));
    };
    auto stage_k = [&](int id) {
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (none[n]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) px[n][i] = __builtin_nanf("");
            }
        put(px, ktile(id), kflag(id), id, false, as_is);
    };
    auto fetch_v = [&](int id) {
        if constexpr (DEEP) fetch(py, vb, rv);
        else fetch(px, vb, rv);
    };
    auto stage_v = [&](int id) {
        const bool edge = key0 + 32 * id + 31 > edge0 || key0 + 32 * id + 32 > key1;
        if constexpr (DEEP) put(py, vtile(id), vflag(id), id, edge, scaled);
        else put(px, vtile(id), vflag(id), id, edge, scaled);
    };
    // Rows: K of tile i is fetched before V of tile i, which takes the rows that K's fetch used.
    __syncthreads();  // the flags
    rows_of(rn, 0);
    fetch_k(0);
    copy_rows(rv, rk);
    stage_k(0);
    fetch_v(0);
    if constexpr (ALT) {
        stage_v(0);
        if constexpr (DEEP) {
            fetch_k(min(1, nsteps - 1));
            copy_rows(rv, rk);
            fetch_v(min(1, nsteps - 1));
        }
    } else if constexpr (DEEP) {
        fetch_k(min(1, nsteps - 1));
    }
    __syncthreads();
    // Half a step behind: the second half's waves meet one barrier more here, the first half's one more at the end.
    if (ALT && w >= NW / 2) __syncthreads();
    for (int id = 0; id < nsteps; ++id) {
        const int k0 = key0 + 32 * id;
        const int n1 = min(id + 1, nsteps - 1), n2 = min(id + 2, nsteps - 1);  // (the last loads itself again, unused)
        const bool active = k0 < kend_w;  // wave-uniform
        const char *const Ks = ktile(id), *const Vs = vtile(id);
        // Phase A: scores and weights; the next K (without ALT: this V) into LDS.
        if constexpr (!DEEP) {
            if constexpr (ALT) {
                fetch_k(n1);
                copy_rows(rv, rk);
            } else {
                fetch_v(id);
            }
        }
        if (active) {
            if constexpr (TREE) windows(tree, k0);
#pragma unroll
            for (int i = 0; i < 2 * NQ; ++i) s[i] = zero4();
            stream_parts<2 * NKS, 3>(
                [&](int i, int part) {
                    return get_row<DP>(Ks, 32, 16 * (i / NKS), 32 * (i % NKS), l16, grp, part);
                },
                [&](int i, auto part, u4 x) {
                    f4 t[NQ];
#pragma unroll
                    for (int n = 0; n < NQ; ++n) t[n] = s[(i / NKS) * NQ + n];
                    mfma_parts<part>(t, x, [&](int n) -> const Tri & { return q[i % NKS][n]; });
#pragma unroll
                    for (int n = 0; n < NQ; ++n) s[(i / NKS) * NQ + n] = t[n];
                });
            const bool kbig = __builtin_amdgcn_readfirstlane(*kflag(id)) == id;
            if (kbig || qbig) {
                // Products with a big operand, from the full values; of both sides, the whole product in f32.
                if (kbig && qbig) {
#pragma unroll
                    for (int i = 0; i < 2 * NQ; ++i) s[i] = zero4();
                }
                const int ll = opaque(lane), lrow = ll & 15, lgrp = ll >> 4;
                const float *krow[2], *qrow[NQ];  // (null: a key without a page, NaN here as where it was staged)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = pool_row(a.pool, table, min(k0 + 16 * j + lrow, key1 - 1));
                    krow[j] = r < 0 ? nullptr : kb + (size_t)r * kld;
                }
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const int r = min(row0 + 16 * n + lrow, rows - 1), t = r / a.G;
                    qrow[n] = a.q + (size_t)(sq.q0 + t) * qld + (size_t)(kvh * a.G + r - t * a.G) * a.dim;
                }
#pragma unroll 1
                for (int cc = 0; cc < 8 * NKS; ++cc) {
                    const int col = 32 * (cc >> 3) + 8 * lgrp + (cc & 7);
                    float kv[2], qv[NQ];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        kv[j] = !krow[j] ? __builtin_nanf("") : FULL || col < a.dim ? krow[j][col] : 0.f;
                        if (!qbig) kv[j] = big_part(kv[j]);
                    }
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        qv[n] = FULL || col < a.dim ? qrow[n][col] * a.scale_log2e : 0.f;
                        if (!kbig) qv[n] = big_part(qv[n]);
                    }
#pragma unroll
                    for (int i = 0; i < 2 * NQ; ++i) s[i] = mfma16(kv[i / NQ], qv[i % NQ], s[i]);
                }
            }
            softmax(k0);
        }
        if constexpr (ALT) {
            stage_k(id + 1);
            if constexpr (DEEP) fetch_k(n2);
        } else {
            stage_v(id);
            if constexpr (DEEP) {
                copy_rows(rv, rk);
                fetch_v(n1);
            }
        }
        __syncthreads();

        // Phase B: the output product; the next V (without ALT: K) into LDS.
        if constexpr (!DEEP) {
            if constexpr (ALT) {
                fetch_v(n1);
            } else {
                fetch_k(n1);
                copy_rows(rv, rk);
            }
        }
        if (active) {
            Tri p[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = s[(i / 4) * NQ + n][i % 4];
                p[n] = split8_as_is(y);
            }
            f4 t[NQ];
            stream_parts<NT, 3>(
                [&](int i, int part) { return get_col<DP>(Vs, 32, 0, 16 * i, lane, part); },
                [&](int i, auto part, u4 x) {
                    if constexpr (part == 0) {
#pragma unroll
                        for (int n = 0; n < NQ; ++n) t[n] = zero4();
                    }
                    mfma_parts<part>(t, x, [&](int n) -> const Tri & { return p[n]; });
                    if constexpr (part == 2) {
#pragma unroll
                        for (int n = 0; n < NQ; ++n) o[i][n] += t[n] * kUnscale1;
                    }
                });
            if (__builtin_amdgcn_readfirstlane(*vflag(id)) == id) {
                // V's big and odd values, from the full rows, to the rows that see them.
                const int ll = opaque(lane), lrow = ll & 15, lgrp = ll >> 4;
                const bool edge = k0 + 31 > edge0 || k0 + 32 > key1;
                if constexpr (TREE) windows(tree, k0);
#pragma unroll 1
                for (int key = 0; key < 32; ++key) {
                    if (k0 + key >= key1) break;
                    const int r = pool_row(a.pool, table, k0 + key);
                    const float *vr = vb + (size_t)max(r, 0) * kld;
                    const int slot = 4 * (key >> 4) + (key & 3);  // of the lane group (key >> 2) & 3
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        unsigned ph = p[n].h.x, pm = p[n].m.x, pl = p[n].l.x;
#pragma unroll
                        for (int e = 1; e < 4; ++e) {
                            ph = slot >> 1 == e ? p[n].h[e] : ph;
                            pm = slot >> 1 == e ? p[n].m[e] : pm;
                            pl = slot >> 1 == e ? p[n].l[e] : pl;
                        }
                        const float pk = __shfl(join_bf16(ph, pm, pl, slot & 1), 16 * ((key >> 2) & 3) + lrow, 64);
                        const bool sees = k0 + key <= last[n] && (!TREE || (tree[n] >> key & 1));
#pragma unroll
                        for (int i = 0; i < NT; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int col = 16 * i + 4 * lgrp + k;
                                if (!sees || (!FULL && col >= a.dim)) continue;
                                const float x = vr[col];
                                if (__builtin_fabsf(x) >= kBig || (edge && x != x)) o[i][n][k] += pk * x;
                            }
                    }
                }
            }
        }
        if constexpr (ALT) {
            stage_v(id + 1);
            if constexpr (DEEP) {
                copy_rows(rv, rk);
                fetch_v(n2);
            }
        } else {
            stage_k(id + 1);
            if constexpr (DEEP) fetch_k(n2);
        }
        __syncthreads();
    }
    if (ALT && w < NW / 2) __syncthreads();

#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int el = opaque(lane), egrp = el >> 4;
        const int r = row0 + 16 * n + (el & 15);
        const float l = sum4grp(lsum[n]);
        if (r >= rows) continue;
        const int t = r / a.G, h = kvh * a.G + r - t * a.G;
        const size_t row = (size_t)(sq.q0 + t);
        if (nch == 1) {
            const float inv = 1.f / l;
            const bool none = TREE && l == 0.f && tree_sees_none(a, (int)row, t, seen0);
            if (egrp == 0) put_stats<TREE>(a, row * a.H + h, m[n], l);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                f4 y = o[i][n] * inv;
                if (none) y = zero4();
                store4(a.out + row * qld + (size_t)h * a.dim, 16 * i + 4 * egrp, a.dim, vec4, y);
            }
        } else {
            const size_t slot = (size_t)sq.at0 + ((size_t)kvh * rows + r) * nch + c;
            if (egrp == 0) { a.part_ml[2 * slot] = m[n]; a.part_ml[2 * slot + 1] = l; }
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if (16 * i + 4 * egrp < a.dim)
                    *reinterpret_cast<f4 *>(a.part_acc + slot * a.part_ld + 16 * i + 4 * egrp) = o[i][n];
        }
    }
}
// Weights of few rows from the scores that the attention stored: of four keys of one
// (sequence, kv head), all rows' added in order.  sp: the keys' scores in row 0; stat(r): row r's base and inverse sum.
// Rows that do not see the keys are skipped (their scores may not be written).
template <class Stat>
DEVI f4 weights_of_few(const float *sp, int kpad, int rows, int G, int seen0, int key, Stat stat) {
    f4 sum = zero4();
    int t = 0, g = 0;
    for (int r = 0; r < rows; ++r) {
        if (key <= seen0 + t) {  // else none of the four keys is seen
            const f4 s = *reinterpret_cast<const f4 *>(sp + (size_t)r * kpad);
            const f2 ml = stat(r);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += key + e <= seen0 + t ? fast_exp2(s[e] - ml.x) * ml.y : 0.f;
        }
        if (++g == G) { g = 0; ++t; }
    }
    return sum;
}
// ---- Merge of the key chunks --------------------------------------------------------
//
// Of one (token, head): M = max_c m_c, out = sum_c acc_c 2^(m_c - M) / sum_c l_c 2^(m_c - M).
// LPR lanes cover a partial row with 16-byte loads.  ROWS false, for few rows of many
// chunks: a workgroup takes a row, each of its 256 / LPR lane groups eight chunks at a time
// (64 chunks at d = 128 take one trip to memory), and the groups are merged in a fixed order; true, for many rows of
// few chunks: each lane group takes a row (65536 rows of 3 chunks at d = 128: 43 us with a wave to a row, 21 so).
// W (with ROWS false): behind a sequence's rows come its weights, 1024 keys of a kv head to a workgroup, which forms
// the rows' statistics from the partials itself instead of waiting for the merge.
template <int DP, bool ROWS, bool W = false, bool TREE = false>
DEVI void paged_merge(const PagedArgs &a) {
    constexpr int LPR = DP <= 32 ? 8 : DP <= 64 ? 16 : DP <= 128 ? 32 : 64, GR = ROWS ? 1 : 256 / LPR;
    constexpr int U = ROWS ? 4 : 8;  // chunks of a lane group in flight
    const int tid = threadIdx.x, g = ROWS ? 0 : tid / LPR, col = 4 * (tid % LPR);
    const int per_wg = ROWS ? 256 / LPR : 1;
    const int item0 = (int)blockIdx.x * per_wg;
    const int item = item0 + (ROWS ? tid / LPR : 0);
    const PagedSeq sq = paged_seq(a.seq, item0);
    // The workgroup's rows, if they are all of one sequence; else each lane group's own.
    int q_len = sq.q_len, n_rows = sq.n_rows, nslots = sq.nch, chunk = sq.chunk, q0 = sq.q0, i = item - sq.first;
    long long at0 = sq.at0;
    if constexpr (ROWS) {
        int k = sq.i;
        while (i >= q_len * a.H) {  // of a sequence behind it, or past the last's end
            if (++k == a.seq.n) return;
            i = item - a.seq.first[k];
            q_len = a.seq.q_len[k]; n_rows = a.seq.n_rows[k]; nslots = a.seq.nch[k]; chunk = a.seq.chunk[k];
            q0 = a.seq.q0[k];
            at0 = a.seq.at0[k];
        }
    }
    const int rows = q_len * a.G;
    if constexpr (W) {
        if (i >= q_len * a.H) {  // workgroup-uniform
            __shared__ f2 stats[32];
            const int per_head = (n_rows + 1023) / 1024, kpad = (n_rows + 15) & ~15, seen0 = n_rows - q_len;
            const int j = i - q_len * a.H, kvh = j / per_head, key = j % per_head * 1024 + 4 * tid;
            const int r = tid >> 3;  // eight threads to a row's chunks
            auto from = [](float m, float to) { return m == -INFINITY ? 0.f : fast_exp2(m - to); };
            float M = -INFINITY, L = 0.f;
            if (r < rows) {
                const float *ml = a.part_ml + 2 * ((size_t)at0 + ((size_t)kvh * rows + r) * nslots);
                const int nch = (seen0 + r / a.G) / chunk + 1;
                for (int c = tid & 7; c < nch; c += 8) {
                    const f2 e = *reinterpret_cast<const f2 *>(ml + 2 * c);
                    const float mb = fmaxf(M, e.x);
                    L = L * from(M, mb) + e.y * from(e.x, mb);
                    M = mb;
                }
            }
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) {
                const float M2 = wave_xor(M, d), L2 = wave_xor(L, d), mb = fmaxf(M, M2);
                L = L * from(M, mb) + L2 * from(M2, mb);
                M = mb;
            }
            if (r < rows && (tid & 7) == 0) stats[r] = f2{M, 1.f / L};
            __syncthreads();
            if (key >= n_rows) return;
            const float *sp = a.scores + a.score0[sq.i] + (size_t)kvh * rows * kpad + key;
            const f4 sum = weights_of_few(sp, kpad, rows, a.G, seen0, key, [&](int x) { return stats[x]; });
            const size_t at = ((size_t)sq.b * a.Hkv + kvh) * a.w_stride + key;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (key + e < n_rows) a.w_out[at + e] = a.w_in[at + e] + sum[e];
            return;
        }
    }
    const int t = i / a.H, h = i % a.H, kvh = h / a.G, r = t * a.G + h % a.G;
    const int nch = (n_rows - q_len + t) / chunk + 1;  // chunks that hold a key the token sees
    const size_t slot0 = (size_t)at0 + ((size_t)kvh * rows + r) * nslots;
    const bool ok = col < a.dim;
    const float *acc = a.part_acc + slot0 * a.part_ld + col;
    const float *ml = a.part_ml + 2 * slot0;
    float M = -INFINITY, L = 0.f;
    f4 A = zero4();
    for (int c0 = U * g; c0 < nch; c0 += U * GR) {
        f2 e[U];
        f4 x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int c = c0 + j;
            const bool in = c < nch;
            e[j] = in ? *reinterpret_cast<const f2 *>(ml + 2 * c) : f2{-INFINITY, 0.f};
            x[j] = in && ok ? *reinterpret_cast<const f4 *>(acc + (size_t)c * a.part_ld) : zero4();
        }
        float mb = M;
#pragma unroll
        for (int j = 0; j < U; ++j) mb = fmaxf(mb, e[j].x);
        const float f0 = M == -INFINITY ? 0.f : fast_exp2(M - mb);
        L *= f0;
        A *= f0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const float f = e[j].x == -INFINITY ? 0.f : fast_exp2(e[j].x - mb);
            L += e[j].y * f;
            A += x[j] * f;
        }
        M = mb;
    }
    if constexpr (!ROWS) {
        __shared__ f4 As[GR][LPR];
        __shared__ f2 Ms[GR];
        const int used = min(GR, (nch + U - 1) / U);  // groups that had a chunk
        if (g < used) As[g][tid % LPR] = A;
        if (g < used && tid % LPR == 0) Ms[g] = f2{M, L};
        __syncthreads();
        if (g != 0) return;
        for (int x = 1; x < used; ++x) M = fmaxf(M, Ms[x].x);
        L = 0.f;
        A = zero4();
        for (int x = 0; x < used; ++x) {
            const f2 y = Ms[x];
            const float f = y.x == -INFINITY ? 0.f : fast_exp2(y.x - M);
            L += y.y * f;
            A += As[x][tid % LPR] * f;
        }
    }
    if (!ok) return;
    const size_t row = (size_t)(q0 + t);
    if (col == 0) put_stats<TREE>(a, row * a.H + h, M, L);
    f4 y = A * (1.f / L);
    if (TREE && L == 0.f && tree_sees_none(a, (int)row, t, n_rows - q_len)) y = zero4();
    store4(a.out + row * a.H * a.dim + (size_t)h * a.dim, col, a.dim, (a.dim & 3) == 0, y);
}
