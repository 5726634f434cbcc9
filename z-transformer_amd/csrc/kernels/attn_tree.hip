// Attention of a tree of drafted tokens over a paged KV cache (gfx950), f32.
//
// A sequence's new tokens, its cache's last rows, are a tree: token t sees the cache's rows before them, and of the new
// tokens those that its mask names, none behind itself:
//     s_j = q_t . k_j / sqrt(d),  out = sum_{j seen} softmax(s)_j v_j,  lse = log sum_j e^{s_j}.
// The products are those of a chunk's attention (attn_paged.h).  Masks are read only by the workgroups, and for the
// tiles, that hold new tokens' keys, one 32-bit window per row and step, which the products of that step hide: the
// rest costs what a chunk's attention does.
#include "attn_paged.h"

// Parents to masks: token t's bits are its own, its parent's, and so on up.  A thread takes a token and goes up to
// the root, from the last word of its mask to the first, so that each word is written once; the way up is a chain of
// reads, out of LDS where the tree fits.  Bound: that chain, and a launch: one tree of 26 tokens 2.2 us, 48 of 61 2.5, 64 of
// 600 5.0; a line of L tokens 0.09 L us (0.18 L from memory, as past 4096 tokens), so that it is better attended as a chunk.
constexpr int kTreeInLds = 4096;
extern "C" __global__ void __launch_bounds__(256) zt_tree_mask(TreeMaskArgs a) {
    __shared__ int up[kTreeInLds];
    const PagedSeq sq = paged_seq(a.seq, blockIdx.x);
    const int t0 = 256 * ((int)blockIdx.x - sq.first), end = min(sq.q_len, t0 + 256);
    const int *parent = a.parent + sq.q0;
    const bool in_lds = end <= kTreeInLds;  // workgroup-uniform
    if (in_lds)
        for (int i = threadIdx.x; i < end; i += 256) up[i] = parent[i];
    __syncthreads();
    const int t = t0 + (int)threadIdx.x;
    if (t >= end) return;
    unsigned long long *row = a.mask + (size_t)(sq.q0 + t) * a.words;
    for (int w = a.words - 1; w > t >> 6; --w) row[w] = 0;
    int depth = 0;
    const auto climb = [&](auto up_of) {
        int w = t >> 6;
        unsigned long long bits = 1ull << (t & 63);
        // Only an earlier token is a parent, so that the way ends.
        for (int at = t, p = up_of(t); p >= 0 && p < at; p = up_of(p)) {
            for (; w > p >> 6; --w) {
                row[w] = bits;
                bits = 0;
            }
            bits |= 1ull << (p & 63);
            ++depth;
            at = p;
        }
        for (; w >= 0; --w) {
            row[w] = bits;
            bits = 0;
        }
    };
    // (Two loops: of one the compiler makes loads through flat addresses for both, 0.15 L us.)
    if (in_lds) climb([&](int i) { return up[i]; });
    else climb([&](int i) { return parent[i]; });
    if (a.pos) a.pos[sq.q0 + t] = sq.n_rows + depth;  // (n_rows: a root's position)
}

#define ZT_TREE_FEW(DP, NQ)                                                                         \
    extern "C" __global__ void __launch_bounds__(256, (DP) == 256 ? 1 : 2) zt_tree_few_d##DP##_n##NQ(PagedArgs a) { \
        paged_few<DP, NQ, true, true>(a);                                                           \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256, (DP) == 256 ? 1 : 2) zt_tree_few_d##DP##_n##NQ##_any(PagedArgs a) { \
        paged_few<DP, NQ, false, true>(a);                                                          \
    }
#define ZT_TREE_MANY(DP, NW, NQ)                                                                    \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_tree_many_d##DP##_##NW##NQ(PagedArgs a) { \
        paged_many<DP, NW, NQ, true, true>(a);                                                      \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(64 * NW, 2) zt_tree_many_d##DP##_##NW##NQ##_any(PagedArgs a) { \
        paged_many<DP, NW, NQ, false, true>(a);                                                     \
    }
#define ZT_TREE(DP)                                                                                 \
    ZT_TREE_FEW(DP, 1)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) zt_tree_merge_d##DP(PagedArgs a) {            \
        paged_merge<DP, false, false, true>(a);                                                     \
    }                                                                                               \
    extern "C" __global__ void __launch_bounds__(256) zt_tree_merge_rows_d##DP(PagedArgs a) {       \
        paged_merge<DP, true, false, true>(a);                                                      \
    }
ZT_TREE(32)
ZT_TREE(64)
ZT_TREE(96)
ZT_TREE(128)
ZT_TREE(192)
ZT_TREE(256)
ZT_TREE_MANY(32, 4, 1) ZT_TREE_MANY(32, 4, 2) ZT_TREE_MANY(32, 8, 2)
ZT_TREE_MANY(64, 4, 1) ZT_TREE_MANY(64, 4, 2) ZT_TREE_MANY(64, 8, 1) ZT_TREE_MANY(64, 8, 2)
ZT_TREE_MANY(96, 4, 1) ZT_TREE_MANY(96, 4, 2) ZT_TREE_MANY(96, 8, 1) ZT_TREE_MANY(96, 8, 2)
ZT_TREE_MANY(128, 4, 1) ZT_TREE_MANY(128, 4, 2) ZT_TREE_MANY(128, 8, 1) ZT_TREE_MANY(128, 8, 2)
ZT_TREE_MANY(192, 4, 1) ZT_TREE_MANY(192, 8, 1)
ZT_TREE_MANY(256, 8, 1)
ZT_TREE_FEW(32, 2) ZT_TREE_FEW(64, 2) ZT_TREE_FEW(96, 2) ZT_TREE_FEW(128, 2)
