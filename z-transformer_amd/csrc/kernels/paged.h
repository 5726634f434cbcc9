// Device-side helpers of the kernels that work on a paged cache.
#pragma once
#include "common.h"
#include "args.h"

// The sequence of a work item, the last whose first item is not past it, and its fields (all
// wave-uniform).  Every field of all sequences is loaded before the item's is known:
// one trip to the arguments instead of two.
struct PagedSeq {
    int i, first, b, q0, q_len, n_rows, nch, chunk;
    long long at0;
};
DEVI PagedSeq paged_seq(const PagedSeqs &s, int item) {
    const int lane = lane_id();
    const int first = s.first[lane], b = s.b[lane], q0 = s.q0[lane], q_len = s.q_len[lane], n_rows = s.n_rows[lane],
              nch = s.nch[lane], chunk = s.chunk[lane];
    const long long at0 = s.at0[lane];
    const int i = __builtin_amdgcn_readfirstlane(
        __popcll(__builtin_amdgcn_ballot_w64(lane < s.n && first <= item)) - 1);
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, i); };
    return {i, of(first), of(b), of(q0), of(q_len), of(n_rows), of(nch), of(chunk),
            (long long)((unsigned long long)(unsigned)of((int)at0) |
                        (unsigned long long)(unsigned)of((int)(at0 >> 32)) << 32)};
}

// Pool row of a sequence's row s, or -1 where its page is none of the pool's.
DEVI int pool_row(const PagePool &p, const int *table, int s) {
    const int page = table[s >> p.shift];
    return (unsigned)page < (unsigned)p.n_pages ? (page << p.shift) + (s & ((1 << p.shift) - 1)) : -1;
}
