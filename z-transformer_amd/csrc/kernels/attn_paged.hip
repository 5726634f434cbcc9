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
// and added to the rows that see them: nothing hidden reaches an output.
#include "common.h"
#include "args.h"
#include "paged.h"

// N consecutive floats (2 or 4) of a row at column c; FULL: the row has DP aligned
// columns; else columns past dim are 0 and rows may be 8-byte aligned only.
template <int N, bool FULL>
DEVI void load_cols(float *dst, const float *row, int c, int dim, bool vec4) {
    if constexpr (N == 4) {
        f4 x = zero4();
        if (FULL || (vec4 && c < dim)) {
            x = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(row + c));
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
        if (FULL || c < dim) x = __builtin_nontemporal_load(reinterpret_cast<const f2 *>(row + c));
        dst[0] = x.x; dst[1] = x.y;
    }
}

// ---- Few rows: K and V stream through registers -----------------------------------
//
// A workgroup takes one (sequence, kv head, chunk of keys, tile of 16 NQ rows); its four waves
// take the chunk's 16-key tiles in turn.  Bound: HBM, each K and V row read once per kv head.
//   * S^T = K Q^T on v_mfma_f32_16x16x4_f32 with the contraction dealt so that k-step
//     (j, e) of lane group grp is column 16 j + 4 grp + e: the A operand is then what
//     lane (l16, grp) loads of key l16 with 16-byte loads, straight from memory.
//   * O^T += V^T P^T in the row-owner layout (common.h): its A operand is what lane
//     (l16, grp) loads of keys 4 grp .. 4 grp + 3, 16 lanes on one row's consecutive chunks.
//   So no byte of K or V passes through LDS, and a row is read in whole 64- and 256-byte pieces.
//   * K of the next tile is loaded when this tile's scores are done, V after its
//     products: one buffer of each, always in flight during the other's half.
template <int DP, int NQ, bool FULL>
DEVI void paged_few(const PagedArgs &a) {
    constexpr int NT = DP / 16, C = ro_chunk<NT>(), NV = NT / C, NW = 4, LW = DP + 4;
    __shared__ float Wacc[NW][16][LW];
    __shared__ float Wm[NW][16], Wl[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sq = paged_seq(a, blockIdx.x);
    const int nch = a.nch[sq], q_len = a.q_len[sq], rows = q_len * a.G;
    int item = (int)blockIdx.x - a.first[sq];
    const int kvh = item % a.Hkv;
    item /= a.Hkv;
    const int c = item % nch, row0 = item / nch * 16 * NQ;
    const int seen0 = a.n_rows[sq] - q_len;  // the cache row of token 0, the last it sees
    const int kend = seen0 + (min(rows, row0 + 16 * NQ) - 1) / a.G + 1;
    const int key0 = c * a.chunk, key1 = min(kend, key0 + a.chunk);
    if (key0 >= kend) return;  // workgroup-uniform
    const int *table = a.pool.table + (size_t)a.b[sq] * a.pool.table_stride;
    const size_t qld = (size_t)a.H * a.dim, kld = (size_t)a.Hkv * a.dim;
    const bool vec4 = (a.dim & 3) == 0;
    const float *kb = a.pool.k + (size_t)kvh * a.dim, *vb = a.pool.v + (size_t)kvh * a.dim;

    // Q: k-step (j, e) is column 16 j + 4 grp + e.  Rows past the last take its values; nothing of them is stored.
    float q[NQ][NT][4];
    int last[NQ];  // the last key that the lane's row sees
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = min(row0 + 16 * n + l16, rows - 1), t = r / a.G;
        last[n] = seen0 + t;
        const float *row = a.q + (size_t)(a.q0[sq] + t) * qld + (size_t)(kvh * a.G + r - t * a.G) * a.dim;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            load_cols<4, FULL>(q[n][j], row, 16 * j + 4 * grp, a.dim, vec4);
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
        for (int j = 0; j < NT; ++j) load_cols<4, FULL>(kx[j], p, 16 * j + 4 * grp, a.dim, vec4);
    };
    auto load_v = [&](int row) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            vrow[r] = __shfl(row, 4 * grp + r, 64);
            const float *p = vb + (size_t)max(vrow[r], 0) * kld;
#pragma unroll
            for (int i = 0; i < NV; ++i) load_cols<C, FULL>(vx[r][i], p, 16 * C * i + C * l16, a.dim, vec4);
        }
    };
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
        const bool edge = k0 + 15 > seen0 || k0 + 16 > key1;  // wave-uniform
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (vrow[r] < 0) s[n][r] = __builtin_nanf("");
                const int key = k0 + 4 * grp + r;
                if (edge && (key > last[n] || key >= key1)) s[n][r] = -INFINITY;
            }
        if (a.scores) {
            const int kpad = (a.n_rows[sq] + 15) & ~15;
            float *sp = a.scores + a.score0[sq] + (size_t)kvh * rows * kpad + k0 + 4 * grp;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int r = row0 + 16 * n + l16;
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
#pragma unroll 1
            for (int key = 0; key < 16; ++key) {
                const int vr = key & 2 ? (key & 1 ? vrow[3] : vrow[2]) : (key & 1 ? vrow[1] : vrow[0]);
                const int row = __shfl(vr, 16 * (key >> 2), 64);
                const float *p = vb + (size_t)max(row, 0) * kld;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float sr = key & 2 ? (key & 1 ? s[n][3] : s[n][2]) : (key & 1 ? s[n][1] : s[n][0]);
                    const float pk = __shfl(sr, 16 * (key >> 2) + l16, 64);
                    const bool sees = k0 + key <= last[n] && k0 + key < key1;
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int col = i / C * 16 * C + C * (4 * grp + r) + i % C;
                            if (!sees || col >= a.dim) continue;
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
            const int i = e / (DP / 4), col = 4 * (e % (DP / 4)), r = row0 + 16 * n + i;
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
            const size_t row = (size_t)(a.q0[sq] + t);
            if (nch == 1) {
                if (col == 0) {
                    const float l2 = M + log2f(L);
                    if (a.lse) a.lse[row * a.H + h] = l2 * 0.69314718055994531f;
                    if (a.stat) a.stat[row * a.H + h] = l2;
                }
                store4(a.out + row * qld + (size_t)h * a.dim, col, a.dim, vec4, A * (1.f / L));
            } else {
                const size_t slot = (size_t)a.part0[sq] + ((size_t)kvh * rows + r) * nch + c;
                *reinterpret_cast<f4 *>(a.part_acc + slot * a.part_ld + col) = A;
                if (col == 0) { a.part_ml[2 * slot] = M; a.part_ml[2 * slot + 1] = L; }
            }
        }
    }
}

// ---- Merge of the key chunks --------------------------------------------------------
//
// A wave takes one (token, head): M = max_c m_c, out = sum_c acc_c 2^(m_c - M) / sum_c l_c 2^(m_c - M).
// LPR lanes cover a partial row with 16-byte loads, 64 / LPR chunks at a time, eight such
// loads in flight; each lane group folds its chunks, then the groups are merged in a fixed order.
template <int DP>
DEVI void paged_merge(const PagedArgs &a) {
    constexpr int LPR = DP <= 32 ? 8 : DP <= 64 ? 16 : DP <= 128 ? 32 : 64, GR = 64 / LPR;
    const int lane = lane_id(), w = threadIdx.x >> 6;
    const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + w);
    const int sq = paged_seq(a, item);
    const int q_len = a.q_len[sq], rows = q_len * a.G, nslots = a.nch[sq];
    const int i = item - a.first[sq];
    if (i >= q_len * a.H) return;  // the last sequence's end
    const int t = i / a.H, h = i % a.H, kvh = h / a.G, r = t * a.G + h % a.G;
    const int nch = (a.n_rows[sq] - q_len + t) / a.chunk + 1;  // chunks that hold a key the token sees
    const size_t slot0 = (size_t)a.part0[sq] + ((size_t)kvh * rows + r) * nslots;
    const int g = lane / LPR, col = 4 * (lane % LPR);
    const bool ok = col < a.dim;
    const float *acc = a.part_acc + slot0 * a.part_ld + col;
    const float *ml = a.part_ml + 2 * slot0;
    float M = -INFINITY, L = 0.f;
    f4 A = zero4();
    for (int c0 = g; c0 < nch; c0 += 8 * GR) {
        float e[8], l[8];
        f4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = c0 + j * GR;
            const bool in = c < nch;
            e[j] = in ? ml[2 * c] : -INFINITY;
            l[j] = in ? ml[2 * c + 1] : 0.f;
            x[j] = in && ok ? *reinterpret_cast<const f4 *>(acc + (size_t)c * a.part_ld) : zero4();
        }
        float mb = M;
#pragma unroll
        for (int j = 0; j < 8; ++j) mb = fmaxf(mb, e[j]);
        const float f0 = M == -INFINITY ? 0.f : fast_exp2(M - mb);
        L *= f0;
        A *= f0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = e[j] == -INFINITY ? 0.f : fast_exp2(e[j] - mb);
            L += l[j] * f;
            A += x[j] * f;
        }
        M = mb;
    }
#pragma unroll
    for (int d = LPR; d < 64; d <<= 1) {  // both sides of an exchange form the same sums
        const float M2 = wave_xor(M, d), mb = fmaxf(M, M2);
        const float f1 = M == -INFINITY ? 0.f : fast_exp2(M - mb), f2v = M2 == -INFINITY ? 0.f : fast_exp2(M2 - mb);
        const bool up = lane & d;
        const float la = L * f1, lb = wave_xor(L, d) * f2v;
        L = up ? lb + la : la + lb;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float xa = A[k] * f1, xb = wave_xor(A[k], d) * f2v;
            A[k] = up ? xb + xa : xa + xb;
        }
        M = mb;
    }
    if (g != 0 || !ok) return;
    const size_t row = (size_t)(a.q0[sq] + t);
    if (col == 0) {
        const float l2 = M + log2f(L);
        if (a.lse) a.lse[row * a.H + h] = l2 * 0.69314718055994531f;
        if (a.stat) a.stat[row * a.H + h] = l2;
    }
    store4(a.out + row * a.H * a.dim + (size_t)h * a.dim, col, a.dim, (a.dim & 3) == 0, A * (1.f / L));
}

// ---- Accumulated weights from stored scores ------------------------------------------
//
// A thread takes four keys of one (sequence, kv head) and adds the weights of all rows,
// rows in order.  Sequences without new tokens copy their weights.
extern "C" __global__ void __launch_bounds__(256) zt_paged_weights(PagedWeightArgs a) {
    const int sq = paged_seq(a, blockIdx.x);
    const int n = a.n_rows[sq], kpad = (n + 15) & ~15, rows = a.q_len[sq] * a.G;
    const int per_head = (n + 1023) / 1024;
    const int item = (int)blockIdx.x - a.first[sq];
    const int kvh = item / per_head, key = (item % per_head) * 1024 + 4 * (int)threadIdx.x;
    if (key >= n) return;
    const float *sp = a.scores + a.score0[sq] + (size_t)kvh * rows * kpad + key;
    const float *st = a.stat + (size_t)a.q0[sq] * a.H + kvh * a.G;
    const int seen0 = n - a.q_len[sq];
    f4 sum = zero4();
    int t = 0, g = 0;
    for (int r = 0; r < rows; ++r) {
        if (key <= seen0 + t) {  // else none of the four keys is seen (and the score may not be written)
            const f4 s = *reinterpret_cast<const f4 *>(sp + (size_t)r * kpad);
            const float l2 = st[(size_t)t * a.H + g];
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += key + e <= seen0 + t ? fast_exp2(s[e] - l2) : 0.f;
        }
        if (++g == a.G) { g = 0; ++t; }
    }
    const size_t at = ((size_t)a.b[sq] * a.Hkv + kvh) * a.w_stride + key;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (key + e < n) a.w_out[at + e] = a.w_in[at + e] + sum[e];
}

#define ZT_PAGED_FEW(DP, NQ)                                                                        \
    extern "C" __global__ void __launch_bounds__(256, 2) zt_paged_few_d##DP##_n##NQ(PagedArgs a) {   \
        paged_few<DP, NQ, true>(a);                                                                 \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256, 2) zt_paged_few_d##DP##_n##NQ##_any(PagedArgs a) { \
        paged_few<DP, NQ, false>(a);                                                                \
    }
#define ZT_PAGED(DP)                                                                                \
    ZT_PAGED_FEW(DP, 1) ZT_PAGED_FEW(DP, 2)                                                         \
    extern "C" __global__ void __launch_bounds__(256) zt_paged_merge_d##DP(PagedArgs a) { paged_merge<DP>(a); }
ZT_PAGED(32)
ZT_PAGED(64)
ZT_PAGED(96)
ZT_PAGED(128)
ZT_PAGED(192)
ZT_PAGED(256)
